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
// whole number of 2^-44. A threshold is found in a histogram over the distance
// from the largest logit, 64 bins to a unit, whose bins that may hold it are
// sorted by one CTA, a token to a thread. top_k counts. For top_p the bins' counts
// give a guess; the exact masses before the bins around it, and of all, are
// then added in registers and theirs in a few counters of each warp (a mass added to
// a histogram costs three atomics, more than the exponential). Where
// the tokens up to top_k's bin are few, that CTA does the rest as well. Bins of too
// many tokens are cut by a second histogram, and what even that leaves crowded
// (many equal logits), or lies beyond its range, is found digit by digit of the
// logits' order keys. All of it is exact and the same on every run.
//
// A row is read once, into the shared memory of a cluster of up to eight CTAs.
//
// Far from bound by HBM (64 rows of 131,072 FP32 logits: 5 us of bytes): a pass
// over the masses is 14 FP64 operations and some fifty instructions a token, one
// over the histogram an atomic. Measured (B200): one row of 32,001, top_k 50 and
// top_p 0.9: 16 us; those 64 rows with top_p 0.95: 78 us, with top_k 50: 38, with
// neither: 37 (two rounds of CTAs, one to an SM: their slices fill its shared
// memory); 256 rows of 50,257 bf16 logits with parameters of their own: 104 us.
// The three passes of digits over counts and masses that the rest falls back to
// took 86, 173 and 173 us.

#include <cooperative_groups.h>

#include "cta_select.cuh"
#include "sample.cuh"

namespace stk {

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 1024, kBins = 1024;  // bins of a histogram: one to a thread
constexpr float kBinsPerUnit = 64.f;
constexpr int kNear = 8;  // bins around the guessed one that are looked at

struct Row {
  float max, half, rate32;  // half of the largest logit
  double top, rate;  // the largest logit, log2 e / T
  double least;      // mass below which a token does not stay
  // Tokens above `limit` stay, of those at it the first `take`.
  uint32_t limit;
  int take;
  // exp((x - max) / T) = 2^t: t = n + f with |f| <= 1/2, 2^f by a polynomial
  // fitted for the least relative error, n added to the exponent. 14 FP64
  // operations, the last of them in_units', bound a pass over the masses.
  __device__ __forceinline__ double mass(float x) const {
    const double d = static_cast<double>(x) - top;
    const double m = fma(d, rate, 6755399441055744.0);  // 1.5 * 2^52: n in the low bits
    const double f = fma(d, rate, 6755399441055744.0 - m);
    double p = fma(f, 1.0148587078171632e-07, 1.325834013445892e-06);
    p = fma(p, f, 1.5252988727215495e-05);
    p = fma(p, f, 0.00015403440864986972);
    p = fma(p, f, 0.0013333557627726357);
    p = fma(p, f, 0.0096181291811879843);
    p = fma(p, f, 0.055504108668400408);
    p = fma(p, f, 0.24022650695722783);
    p = fma(p, f, 0.69314718055988556);
    p = fma(p, f, 1.0);
    const double e = __hiloint2double(__double2hiint(p) + (__double2loint(m) << 20), __double2loint(p));
    // Nothing below 2^-60, nor of -inf at an infinite temperature (no number); infinities weigh alike.
    // (Half the distance: the whole one may pass FP32's largest number.)
    return x == max ? 1.0 : fmaf(x, -0.5f, half) * rate32 <= 30.f ? e : 0.0;
  }
  // As a whole number of 2^-44: the last bits of e + 256.
  static __device__ __forceinline__ u64 in_units(double e) {
    return static_cast<u64>(__double_as_longlong(e + 256.0) - __double_as_longlong(256.0));
  }
  // 0 for a token of too little mass.
  __device__ __forceinline__ u64 units(float x) const {
    const double e = mass(x);
    return e >= least ? in_units(e) : 0ull;
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
  float best;  // of the CTA: the largest logit
  int token;   // and the lowest token that has the row's
  int warp_min[32];
  uint32_t part_low[32][2 * kNear + 1], part_high[32][2 * kNear + 1];  // mass of each warp's stretch in each of the bins that may hold the threshold
  double warp_doubles[32];
  int from;          // the bin that is guessed to hold the threshold
  u64 whole;         // mass of all tokens
  double bound, last;
  int equal;   // tokens at the limit
  u64 sum;     // mass of what stays
  int listed;  // tokens asked into the list
  int owned;   // and into the CTA's own
  int bin;
  u64 above;         // of the goal, before the bin
  int upto, crowd;   // tokens up to the bin, and in it
  uint32_t limit;  // the threshold found
  int take;
};

__device__ __forceinline__ void add_mass(uint32_t* low, uint32_t* high, u64 e) {
  const uint32_t e_low = static_cast<uint32_t>(e), old = atomicAdd(low, e_low);
  const uint32_t e_high = static_cast<uint32_t>(e >> 32) + (old + e_low < old ? 1u : 0u);
  if (e_high) atomicAdd(high, e_high);
}
__device__ __forceinline__ void add_mass(Hist& h, int bin, u64 e) { add_mass(&h.low[bin], &h.high[bin], e); }

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
  float best = neg_inf();  // (fmaxf passes NaN over)
  int done = 0;
  if (reinterpret_cast<uintptr_t>(src) % 16 == 0) {
    done = n / kVec * kVec;
#pragma unroll 8
    for (int i = tid * kVec; i < done; i += kThreads * kVec) {
      const uint4 v = *reinterpret_cast<const uint4*>(src + i);
      *reinterpret_cast<uint4*>(row + i) = v;
      const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
      for (int j = 0; j < kVec; ++j) best = fmaxf(best, to_f32(e[j]));
    }
  }
#pragma unroll 8
  for (int i = done + tid; i < n; i += kThreads) {
    const T v = src[i];
    row[i] = v;
    best = fmaxf(best, to_f32(v));
  }
  for (int i = tid; i < kBins; i += kThreads) sh.hist.count[i] = sh.hist.low[i] = sh.hist.high[i] = 0;
  if (tid == 0) sh.listed = sh.owned = 0;
  best = warp_max(best);
  if (lane == 0) sh.warp_doubles[warp] = best;
  __syncthreads();
  best = warp_max(static_cast<float>(sh.warp_doubles[lane]));
  if (tid == 0) sh.best = best;
  cluster.sync();
  for (int p = 0; p < parts; ++p) best = fmaxf(best, *cluster.map_shared_rank(&sh.best, p));
  const float temperature = a.temperature.rows ? a.temperature.rows[r] : a.temperature.all;
  const bool nothing = best == neg_inf();
  if (nothing || !(temperature > 0.f)) {
    // ---- greedy: the lowest token with the largest logit
    int token = 0x7fffffff;
    if (!nothing)
      all_tokens([&](int i, float x) {
        if (x == best) token = min(token, begin + i);
      });
    token = __reduce_min_sync(kFull, token);
    if (lane == 0) sh.warp_min[warp] = token;
    __syncthreads();
    token = __reduce_min_sync(kFull, sh.warp_min[lane]);
    if (tid == 0) sh.token = token;
    cluster.sync();
    if (part == 0) {
      for (int p = 0; p < parts; ++p) token = min(token, *cluster.map_shared_rank(&sh.token, p));
      if (tid == 0) a.tokens[r] = nothing ? -1 : token;
      if (tid == 0 && nothing) report(a.status, kStatusNoToken);
    }
    cluster.sync();  // the first CTA has read
    return;
  }
  Row w;
  w.max = best;
  w.half = 0.5f * best;
  w.top = static_cast<double>(best);
  w.rate = 1.4426950408889634 / static_cast<double>(temperature);
  w.rate32 = static_cast<float>(w.rate);
  w.least = 0.0;
  w.limit = 0;
  w.take = 0x7fffffff;  // (all above)
  const int top_k = a.top_k.rows ? a.top_k.rows[r] : a.top_k.all;
  const float top_p = a.top_p.rows ? a.top_p.rows[r] : a.top_p.all;
  const float min_p = a.min_p.rows ? a.min_p.rows[r] : a.min_p.all;

  // f(i, logit, mass) for a stretch's tokens; the masses of several are computed side by side, whether they are used or
  // not (one after the other, behind a branch, each waits for its chain of FP64 products: three times as long).
  auto with_masses = [&](int from, int to, auto f) {
    int i = from + lane * kVec;
    for (; i + kVec <= to; i += 32 * kVec) {
      const uint4 v = *reinterpret_cast<const uint4*>(row + i);
      const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
      for (int j = 0; j < kVec; j += 4) {
        float x[4];
        double m[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) x[q] = clean(to_f32(e[j + q]));
#pragma unroll
        for (int q = 0; q < 4; ++q) m[q] = w.mass(x[q]);
#pragma unroll
        for (int q = 0; q < 4; ++q) f(i + j + q, x[q], m[q]);
      }
    }
    for (; i < to; ++i) {
      const float x = logit(i);
      f(i, x, w.mass(x));
    }
  };
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

  // The bin of a logit: its distance from the largest, rounded to whole bins (by adding 2^23); the last has no end.
  auto coarse_bin = [&](float x) {
    const float d = fminf(x == w.max ? 0.f : w.max - x, static_cast<float>(kBins - 1) / kBinsPerUnit);
    return __float_as_int(fmaf(d, kBinsPerUnit, 8388608.f)) - 0x4b000000;
  };
  u64* list = cluster.map_shared_rank(sh.list, 0);
  int* listed = cluster.map_shared_rank(&sh.listed, 0);
  // Tokens into the first CTA's list: first into an own one (over the histogram, which is clear before and after).
  u64* own = reinterpret_cast<u64*>(&sh.hist);
  auto enlist = [&](int i, uint32_t key) {
    const int at = atomicAdd(&sh.owned, 1);
    if (at < kThreads) own[at] = static_cast<u64>(key) << 32 | static_cast<uint32_t>(~(begin + i));
  };
  auto hand_over = [&]() {
    __syncthreads();
    const int m = min(sh.owned, kThreads);
    if (tid == 0) sh.bin = atomicAdd(listed, sh.owned);
    __syncthreads();
    if (tid < m && sh.bin + tid < kThreads) list[sh.bin + tid] = own[tid];
    __syncthreads();
    if (tid == 0) sh.owned = 0;
    sh.hist.count[tid] = sh.hist.low[tid] = sh.hist.high[tid] = 0;
    cluster.sync();
  };
  // Each warp's stretch of the slice.
  const int stretch = (n + 32 * 32 - 1) / (32 * 32) * 32, w0 = min(n, warp * stretch), w1 = min(n, w0 + stretch);
  // In the first CTA: of its sorted list's m tokens, the thread's one weighs v; the one that reaches the goal sets the
  // threshold. `partly`: of its logit do not all tokens stay that could.
  auto set_limit = [&](uint32_t key, int same, bool partly) {
    // The last of its logit: all of that logit stay, and need not be told apart.
    sh.limit = partly ? key : key - 1;
    sh.take = partly ? same + 1 : 0x7fffffff;
  };
  auto sorted = [&](int m) {  // the list in descending order; the thread's token, and its place among those of its logit
    u64 x = tid < m ? sh.list[tid] : 0;
    x = sort_descending(x, m, sh.list);
    __syncthreads();
    sh.list[tid] = x;
    __syncthreads();
    const uint32_t key = static_cast<uint32_t>(x >> 32);
    int first = tid, lo = 0;  // the first place with the key
    while (tid < m && lo < first) {
      const int mid = (lo + first) >> 1;
      if (static_cast<uint32_t>(sh.list[mid] >> 32) > key) lo = mid + 1; else first = mid;
    }
    return make_uint2(key, static_cast<uint32_t>(tid - first));
  };
  auto last_of_logit = [&](int m, uint32_t key) { return tid + 1 == m || static_cast<uint32_t>(sh.list[tid + 1] >> 32) != key; };

  // Of the cluster's histograms, the thread's bin (in the order of descending logits).
  auto cluster_bin = [&](int bin, u64& count, u64& mass, bool masses) {
    count = mass = 0;
    for (int p = 0; p < parts; ++p) {
      const Hist* h = cluster.map_shared_rank(&sh.hist, p);
      count += h->count[bin];
      if (masses) mass += static_cast<u64>(h->high[bin]) << 32 | h->low[bin];
    }
  };
  auto clear = [&]() {  // once all have read
    cluster.sync();
    sh.hist.count[tid] = sh.hist.low[tid] = sh.hist.high[tid] = 0;
    __syncthreads();
  };

  // ---- top_p alone: a guess from the bins' counts, then the exact masses around it
  bool narrow = false;        // the bins that may hold it are few, and each warp knows their masses in its stretch
  bool before_known = false;  // the mass of what stays of the stretch in the bins before `from`
  u64 before_mass = 0;
  int from = 0, to = 0;
  const bool searched = (top_k <= 0 || top_k >= a.V) && top_p < 1.f;
  bool decided = false;       // top_p leaves all that min_p does
  u64 count = 0;              // tokens of the thread's bin
  if (searched) {
    all_tokens([&](int, float x) { atomicAdd(&sh.hist.count[coarse_bin(x)], 1u); });
    cluster.sync();
    u64 none;
    cluster_bin(tid, count, none, false);
    // Were all of a bin at its middle, the threshold would be in bin `guess`; the masses within bins are even enough that
    // it is at most a few bins away (if not, it is searched for below).
    const double about = count ? static_cast<double>(count) * exp2(-tid / static_cast<double>(kBinsPerUnit) * w.rate) : 0.0;
    double all_about;
    const double up_to = scan_add<double>(about, sh.warp_doubles, all_about) + about;
    const double share = top_p > 0.f ? static_cast<double>(top_p) : 0.0;
    if (tid == 0) sh.from = kBins - 1;
    __syncthreads();
    const int guess = __reduce_min_sync(kFull, up_to >= share * all_about ? tid : kBins - 1);
    if (lane == 0) atomicMin(&sh.from, guess);
    __syncthreads();
    from = max(0, sh.from - kNear);
    to = min(kBins - 1, sh.from + kNear);
    // min_p decides alone where everything before `from` surely stays by top_p and nothing from there on does by min_p: a
    // mass is off its bin's middle by half a bin and what rounding moves a distance by.
    const double bar = min_p > 0.f ? fmin(static_cast<double>(min_p), 1.0) : 0.0;
    const double half = 0.5 / kBinsPerUnit + 4e-6, factor = exp2(half * w.rate);
    if (tid == max(from, 1) - 1) sh.bound = up_to;
    if (tid == kBins - 1) sh.last = about;
    __syncthreads();
    decided = from > 0 && exp2(-(from / static_cast<double>(kBinsPerUnit) - half) * w.rate) < bar * (1 - 1e-9) &&
              sh.bound * factor * factor < share * (all_about - sh.last) * (1 - 1e-6);
    if (decided) clear();
  }
  if (searched && !decided) {
    const double bar = min_p > 0.f ? fmin(static_cast<double>(min_p), 1.0) : 0.0;
    const double share = top_p > 0.f ? static_cast<double>(top_p) : 0.0;
    // ---- the exact mass of all, of the bins before, and of each that may hold the threshold
    u64 whole = 0, above = 0;
    narrow = bar == 0.0;
    if (narrow) {  // by warps as well, whose stretches' masses need no second look then
      if (lane <= 2 * kNear) sh.part_low[warp][lane] = sh.part_high[warp][lane] = 0;
      __syncwarp();
      with_masses(w0, w1, [&](int, float x, double m) {
        const int bin = coarse_bin(x);
        const u64 e = Row::in_units(m);
        whole += e;
        above += bin < from ? e : 0ull;
        if (bin >= from && bin <= to) add_mass(&sh.part_low[warp][bin - from], &sh.part_high[warp][bin - from], e);
      });
      before_mass = above;
      __syncthreads();
      if (tid <= to - from) {
        u64 e = 0;
        for (int i = 0; i < 32; ++i) e += static_cast<u64>(sh.part_high[i][tid]) << 32 | sh.part_low[i][tid];
        sh.hist.low[from + tid] = static_cast<uint32_t>(e);
        sh.hist.high[from + tid] = static_cast<uint32_t>(e >> 32);
      }
    } else {
      with_masses(w0, w1, [&](int, float x, double m) {
        const int bin = coarse_bin(x);
        const u64 e = Row::in_units(m), early = bin < from ? e : 0ull;
        whole += e;
        above += early;
        before_mass += m >= bar ? early : 0ull;
        if (bin >= from && bin <= to) add_mass(sh.hist, bin, e);
      });
    }
    u64 total;
    scan_add<u64>(whole, sh.warp_sums, total);
    if (tid == 0) sh.whole = total;
    scan_add<u64>(above, sh.warp_sums, total);
    if (tid == 0) sh.sum = total;
    cluster.sync();
    whole = above = 0;
    for (int p = 0; p < parts; ++p) {
      whole += *cluster.map_shared_rank(&sh.whole, p);
      above += *cluster.map_shared_rank(&sh.sum, p);
    }
    // The least whole number that is not below top_p of the mass; the first token always stays.
    u64 goal = static_cast<u64>(ceil(share * static_cast<double>(whole)));
    goal = goal < 1 ? 1 : goal > whole ? whole : goal;
    u64 again, mass;
    cluster_bin(tid, again, mass, true);
    if (tid == 0) sh.crowd = kThreads + 1;
    const u64 before = above + scan_add<u64>(mass, sh.warp_sums, total);
    if (tid >= from && tid <= to && before < goal && before + mass >= goal) {
      sh.bin = tid;
      sh.above = before;
      sh.crowd = static_cast<int>(count);
    }
    clear();
    const int bin = sh.bin;
    if (sh.crowd <= kThreads) {
      // ---- the bin's tokens, sorted by the first CTA
      all_tokens([&](int i, float x) {
        if (coarse_bin(x) == bin) enlist(i, order_key(x));
      });
      hand_over();
      if (part == 0) {
        const int m = sh.listed;
        const uint2 at = sorted(m);
        const u64 v = tid < m ? w.units(value_of(at.x)) : 0;
        const u64 up_to = sh.above + scan_add<u64>(v, sh.warp_sums, total);
        if (up_to < goal && up_to + v >= goal) set_limit(at.x, static_cast<int>(at.y), !last_of_logit(m, at.x));
        if (tid == 0) sh.listed = 0;
      }
      cluster.sync();
      w.limit = *cluster.map_shared_rank(&sh.limit, 0);
      w.take = *cluster.map_shared_rank(&sh.take, 0);
      before_known = true;
      to = bin;
    }
  }

  // ---- thresholds: first by counts (top_k), then by masses (top_p)
  for (int mode = 0; mode < 2; ++mode) {
    const bool counts = mode == 0;
    if (counts ? top_k <= 0 || top_k >= a.V : !(top_p < 1.f) || before_known || decided) continue;
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
        const int bin = coarse_bin(x);
        if (level == 0) return bin;
        const float d = x == w.max ? 0.f : w.max - x;
        const float in = (d - (static_cast<float>(crowded) - 0.5f) / kBinsPerUnit) * (kBinsPerUnit * kBins);
        return bin != crowded ? -1 : static_cast<int>(fminf(fmaxf(in, 0.f), static_cast<float>(kBins - 1)));
      };
      all_tokens([&](int, float x) {
        const int bin = bin_of(x);
        if (bin >= 0) weigh(x, order_key(x), bin);
      });
      if (some_at_limit && bin_of(value_of(w.limit)) >= 0) weigh_limit(bin_of(value_of(w.limit)));
      cluster.sync();
      u64 count, mass;
      cluster_bin(tid, count, mass, !counts);
      choose(count, mass, level == 0);
      const int bin = sh.bin, crowd = sh.crowd, upto = sh.upto;
      clear();
      if (level == 0 && upto <= kThreads && !some_at_limit) {
        // ---- few: all of them (those that top_k left: `upto` counts no others) go to the first CTA, which does the rest
        all_tokens([&](int i, float x) {
          const uint32_t key = order_key(x);
          if (bin_of(x) <= bin && (counts || key > w.limit)) enlist(i, key);
        });
        hand_over();
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
      hand_over();
      if (part == 0) {
        const int m = sh.listed;
        if (m <= kThreads) {  // (more where some at top_k's limit do not stay)
          const uint2 at = sorted(m);
          const int same = static_cast<int>(at.y);
          u64 v = 0;
          if (tid < m && !(some_at_limit && at.x == w.limit && same >= w.take)) v = counts ? 1ull : w.units(value_of(at.x));
          u64 total;
          const u64 before = scan_add<u64>(v, sh.warp_sums, total);
          if (before < goal && before + v >= goal)
            set_limit(at.x, same, (some_at_limit && at.x == w.limit) || !last_of_logit(m, at.x));
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
      cluster_bin(tid, count, mass, !counts);
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
  // Mass of a token, with `e` tokens at the limit before it. (Without ties the limit is the order key below the last
  // logit that stays: a logit one unit in its last place lower does not.)
  auto stays = [&](float x, int e) {
    const uint32_t key = order_key(x);
    return key > w.limit || (ties && key == w.limit && e < w.take) ? w.units(x) : 0ull;
  };
  u64 sum = 0;
  if (before_known && !ties) {
    sum = before_mass;
    if (narrow) {
      if (lane < to - from) sum += static_cast<u64>(sh.part_high[warp][lane]) << 32 | sh.part_low[warp][lane];
      for_each(w0, w1, lane, 32, [&](int, float x) {
        if (coarse_bin(x) == to && order_key(x) > w.limit) sum += w.units(x);
      });
    } else with_masses(w0, w1, [&](int, float x, double m) {
      const int bin = coarse_bin(x);
      const bool in = (static_cast<unsigned>(bin - from) <= static_cast<unsigned>(to - from)) & (order_key(x) > w.limit) &
                      (m >= w.least);
      sum += in ? Row::in_units(m) : 0ull;
    });
  } else if (!ties) {
    with_masses(w0, w1, [&](int, float x, double m) {
      sum += (order_key(x) > w.limit) & (m >= w.least) ? Row::in_units(m) : 0ull;
    });
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
  // CTAs of a row: as many as its logits need, more while they find SMs and 16 K logits each. One FP32 row of 32,001
  // takes 16.4 us by the two CTAs of this rule (by one 20.5, four 14.4, eight 14.4 to 17.0) with top_k 50 and top_p 0.9,
  // 28.7 (36.9, 24.6, 25.5) with top_p 0.95 alone; one of 131,072 33 to 34 by its eight (39 by four).
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
