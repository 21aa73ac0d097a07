// Attention weight received by each cached key, on the tensor cores (tcgen05).
//
// The sum over rows (new tokens x query heads of the group) of 2^(c s - lse) is
// taken per key, so S is formed with the keys along the tensor memory's lanes:
//   S^T = K Q^T        128 keys x up to 112 rows, FP32 in tensor memory
//   sum += 2^(c S - lse)   one thread per key; a row's log-sum-exp, known
//                          beforehand, is the same for all of a warp's keys
// No running maximum, no sums across lanes: a key's sum is taken in the order of
// its rows, and reaches the weights by one reduction, the key's only one.
//
// A job is 256 keys (128 where the rows are few) of one request's KV head and a
// part of its rows. The CTAs of a persistent grid (one per SM) take the jobs in
// turn; copies run ahead of the products across the borders of jobs, the next
// job's K under the current one's rows. With single tokens K streams through a
// ring of six tiles, with prompts the row tiles do, one in shared memory for
// both halves of the keys (a tile from L2 serves 256 x 112 scores: half of
// what 128 keys would ask of L2). Parts of the rows have sums of their own,
// which a second kernel adds in order.
//
// Warps 0-15 (0-3 for few rows): exponentials and sums. Four take an MMA tile's
// 128 keys; where the rows are many two such groups take every second row tile,
// so that one's waits run under the other's exponentials, and add up at a job's
// end. Then one warp for the MMAs, two for the copies (TMA; K and Q, or with few
// rows every second job), one that walks over jobs and row tiles ahead of all
// others, and four for the log-sum-exps and key intervals of the row tiles'
// rows, in turn.
//
// HBM-bound for single tokens: K is read once. 64 requests of 8-32 K tokens, 16 /
// 8 heads, bf16 (2.6 GB): 396 us, 6.7 TB/s; 16 requests of 4-12 K: 49 us, 80 %
// of a copy's rate. What it took: whole pages of a head in one copy each (a
// 5-dimensional map puts the halves of 8 keys next to each other), issued as
// predicates of uniform code (128-dim boxes lane by lane cost 130 clocks each
// and held the kernel at 58 %), and results added by reductions that nobody
// waits for.
//
// With prompts bound by the exponentials in principle: 16 per SM and clock, 1,792
// clocks for 256 keys x 112 rows, whose products are 960. In fact about 3,000:
// a warp's waits and the tile's bookkeeping, some 1,100 clocks, run under the
// other group's exponentials only in part. Three prompts of 1.5-8 K tokens, 16 / 8
// heads, D 128: 180 us (69 at the tensor cores' rate), capped 261; the last 64
// tokens of 4 prompts of 17-32 K: 102; 15 K tokens in a window of 1,024, D 64,
// biased: 339. On the plain prompts, in the order tried: every load warp
// walking over all items 194-243 us, one walking warp 194, batches of its row tiles
// 184, row tiles by turns instead of halves of each 180; row tiles of 64 with four
// S buffers 199, exponentials on the FMA units 188-228 (the issue slots, not the
// special function unit alone, are short), waits with long suspensions 241.
//
// Rows that see none of a warp's keys are skipped tile by tile, tiles whose
// rows all see all of a warp's keys need no mask. Unseen keys may hold
// anything: each key is a lane of its own, selected, never multiplied. Boxes
// of keys that no row of the job sees are not looked up and read as zeros.
// Rows that only fill up the MMA's sixteens are left out of the sums, by kernels
// of their own (drafts of 5 tokens of 4 heads: 64 us with them, NaN at infinite
// keys, 68.5 without; where more tokens fit into these rows there are none).

#include "paged_tensor.cuh"
#include "tcgen05.cuh"
#include "weigh.cuh"

namespace stk {

int set_wait_limit_weigh(unsigned long long ns) { return set_wait_limit_this_unit(ns); }

namespace {

constexpr int kInfoWarps = 4, kCopyWarps = 2;
constexpr int kRun = 16;  // rows taken from tensor memory at once

// Keys that a row tile's rows see: least and end of any row's, of all rows'.
struct Range {
  int any_lo, any_hi, all_lo, all_hi;
};

// Up to 32 row tiles of a job, as the walk hands them on.
struct alignas(16) Batch {
  int h, k0, part;       // job: KV head, first key, part of the request's rows
  int room;              // keys from k0 on that are there
  int first, last;       // batch of the job
  int stop;
  unsigned mask;         // row tiles tile + i; none: a job of which only the zeros are to be written
  int block0;            // the request: first block, new tokens, tokens in the cache, tokens weighed
  int t0, n_all, len;
  int n, tile;
  int keys_lo, keys_hi;  // that the part's rows see
  int q, k;              // row tiles and K tiles copied before it
};

// A row tile of a job, as the products and sums take it.
struct alignas(16) Item {
  int h, k0, part, room;
  int first, last, empty, stop;
  Range range;
  int block0;
};

template <int ROWS, int KEYS>
struct Info {
  Item item;
  alignas(16) float neg_lse[ROWS];   // - log-sum-exp * log2 e
  alignas(16) float2 bias[ROWS];     // slope * log2 e, place
  alignas(16) int2 keys[ROWS];       // lo, hi
  float other[KEYS > 128 ? KEYS : 1];  // sums of the second group's rows, at a job's end
};

template <int D, bool FEW>
struct Plan {
  static constexpr int kTiles = FEW ? 1 : 2;        // MMA tiles of a job
  static constexpr int kKeys = 128 * kTiles, kRows = FEW ? kWeighFew : kWeighRows;
  static constexpr int kKBytes = kKeys * D * 2;  // 8 keys of 64 dims after 8 keys of 64 dims, 1,024 bytes each
  static constexpr int kQBytes = kRows * D * 2, kQHalf = kRows * 128;
  static constexpr int kKRing = FEW ? (D == 128 ? 6 : 10) : 2;
  static constexpr int kQRing = FEW ? 4 : D == 128 ? 3 : 6;
  static constexpr int kInfos = FEW ? 8 : 4;        // row tiles whose rows' data are held
  static constexpr int kAhead = FEW ? 8 : 4;        // batches that the walk is ahead
  static constexpr int kBuffers = FEW ? 4 : 2;      // S in tensor memory
  static constexpr int kBufferCols = FEW ? 16 : 256, kTmem = kBuffers * kBufferCols;
  static constexpr int kGroups = FEW ? 1 : 2;
  static constexpr int kSumWarps = 4 * kTiles * kGroups, kThreads = (kSumWarps + 2 + kCopyWarps + kInfoWarps) * 32;
  static_assert(kInfos % kInfoWarps == 0 && (!FEW || (kKRing % kCopyWarps == 0 && kQRing % kCopyWarps == 0)),
                "each slot is filled by one warp");
};

template <int D, bool FEW>
struct Shared {
  using P = Plan<D, FEW>;
  alignas(1024) unsigned char k[P::kKRing][P::kKBytes];
  alignas(1024) unsigned char q[P::kQRing][P::kQBytes];
  Info<P::kRows, P::kKeys> info[P::kInfos];
  Batch ahead[P::kAhead];
  uint64_t k_full[P::kKRing], k_empty[P::kKRing];
  uint64_t q_full[P::kQRing], q_empty[P::kQRing];
  uint64_t i_full[P::kInfos], i_empty[P::kInfos], i_other[P::kInfos];
  uint64_t w_full[P::kAhead], w_empty[P::kAhead];
  uint64_t s_full[P::kBuffers][2], s_empty[P::kBuffers][2];
  uint64_t drained;
  volatile int k_asked[kCopyWarps], q_asked[kCopyWarps];  // copies asked for, by each of the warps that ask
  uint32_t tmem;
};

// D = A B by one elected lane, from the descriptors' halves: the lower ones
// differ, the upper ones are the call's.
__device__ __forceinline__ void mma_halves(uint32_t d, uint32_t a, uint32_t a_hi, uint32_t b, uint32_t b_hi, uint32_t idesc,
                                           bool acc) {
  asm volatile(
      "{\n .reg .pred p, e;\n .reg .b64 x, y;\n mov.b64 x, {%1, %2};\n mov.b64 y, {%3, %4};\n setp.ne.u32 p, %6, 0;\n"
      " elect.sync _|e, 0xffffffff;\n @e tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %5, p;\n}\n" ::"r"(d),
      "r"(a), "r"(a_hi), "r"(b), "r"(b_hi), "r"(idesc), "r"(static_cast<uint32_t>(acc))
      : "memory");
}

// Copies by one elected lane, as predicates inside warp-uniform code (under a
// branch, or with operands by lane, one takes over a hundred clocks).
__device__ __forceinline__ void tma_keys(const CUtensorMap* map, uint32_t dst, uint32_t bar, int y, int page_head) {
  asm volatile(
      "{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n"
      " @e cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %3, %3, %4, %5}], "
      "[%2];\n}\n" ::"r"(dst),
      "l"(map), "r"(bar), "r"(0), "r"(y), "r"(page_head)
      : "memory");
}
__device__ __forceinline__ void tma_rows(const CUtensorMap* map, uint32_t dst, uint32_t bar, int x, int head, int token) {
  asm volatile(
      "{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n"
      " @e cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], "
      "[%2];\n}\n" ::"r"(dst),
      "l"(map), "r"(bar), "r"(x), "r"(head), "r"(token), "r"(0)
      : "memory");
}

// The request r as it is weighed: its new tokens and its row tiles.
struct Rows {
  RowTile t;
  int n, tiles;  // tokens (at most w.most), row tiles
};

__device__ __forceinline__ Rows rows_of(const WeighArgs& w, int r) {
  const PagedAttnArgs& a = w.a;
  Rows x;
  const int2 tn = new_tokens(a.token_offsets, r, a.R, a.T, a.status);
  x.t.r = r;
  x.t.row0 = x.t.rows = 0;
  x.t.t0 = tn.x;
  x.t.n = tn.y;
  x.t.len = tn.y > 0 ? cached_tokens(a, r, tn.y) : 0;
  x.n = min(tn.y, w.most);
  if (tn.y > w.most) report(a.status, kStatusShapeOverflow);
  x.tiles = (x.n + w.tokens - 1) / w.tokens * w.head_parts;
  return x;
}

__device__ __forceinline__ int parts_of(const WeighArgs& w, const Rows& x) { return (x.tiles + w.per_part - 1) / w.per_part; }

// The keys [.x, .y) that any row of part p of a request sees.
__device__ __forceinline__ int2 part_keys(const WeighArgs& w, const Rows& x, int p) {
  if (w.part_keys) return w.part_keys[static_cast<long long>(x.t.r) * w.parts + p];
  const int tiles = min(x.tiles, (p + 1) * w.per_part);
  const int tokens = min(x.n, ((tiles - 1) / w.head_parts + 1) * w.tokens);
  return make_int2(0, max(0, min(x.t.len - x.t.n + tokens, x.t.len)));
}

// Key tiles of a part: first and number.
template <int KEYS>
__device__ __forceinline__ int2 part_tiles(const WeighArgs& w, const Rows& x, int p) {
  const int2 k = part_keys(w, x, p);
  if (k.x >= k.y) return make_int2(0, 0);
  return make_int2(k.x / KEYS, (k.y + KEYS - 1) / KEYS - k.x / KEYS);
}

// Keys that tokens [i, i + w.tokens) of a request see under the causal mask.
__device__ __forceinline__ Range causal_range(const WeighArgs& w, const Rows& x, int i) {
  const int pos = x.t.len - x.t.n + i, last = min(w.tokens, x.n - i) - 1;
  Range g;
  g.any_lo = g.all_lo = 0;
  g.any_hi = max(0, min(pos + last + 1, x.t.len));
  g.all_hi = max(0, min(pos + 1, x.t.len));
  return g;
}

// Keys that a chunk of a request's tokens sees.
__device__ __forceinline__ Range range_of(const WeighArgs& w, const Rows& x, int chunk) {
  if (w.ranges == nullptr) return causal_range(w, x, chunk * w.tokens);
  const int4 g = w.ranges[weigh_range_at(x.t.t0, x.t.r, w.tokens) + chunk];
  return Range{g.x, g.y, g.z, g.w};
}

// The walk over the CTA's jobs and their row tiles, by one warp. FEW: every
// request is one row tile, one part.
template <int KEYS, bool FEW>
struct Walk {
  // a window of 32 requests, one per lane
  int r0, base;          // base: first block of the lane's request
  Rows mine;
  int2 whole;            // key tiles of its only part (w.parts = 1)
  int2 seen_keys;        // keys of its only part (FEW)
  long long end, total, before;  // jobs up to the lane's request, of the window, before the window
  long long job;         // of all
  int in_run;
  // the current request and its parts, one per lane: first key tile, key tiles up to it
  Rows x;
  int block0, part_first, part_end;
  long long x_begin, x_end;  // its jobs, within the window
  // the current job
  int h, k0, part;
  int2 keys;             // that the part's rows see
  int w0, qb;            // its next 32 row tiles, end of its row tiles
  unsigned seen;         // those that see a key of the job
  bool started;
  int n_q, n_k;

  __device__ __forceinline__ void window(const WeighArgs& w, int lane) {
    const int r = r0 + lane;
    mine = Rows{};
    base = 0;
    end = 0;
    if (r < w.a.R) {
      mine = rows_of(w, r);
      base = w.a.L.block_offsets[r];
      const int parts = parts_of(w, mine);
      for (int p = 0; p < parts; ++p) {
        whole = part_tiles<KEYS>(w, mine, p);
        end += whole.y;
      }
      end *= w.a.L.hkv;
      if (FEW && mine.n > 0) seen_keys = part_keys(w, mine, 0);
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(kFull, end, o);
      if (lane >= o) end += y;
    }
    total = __shfl_sync(kFull, end, 31);
  }

  __device__ __forceinline__ void start(const WeighArgs& w, int lane) {
    r0 = 0;
    before = 0;
    started = false;
    whole = make_int2(0, 0);
    x_begin = x_end = 0;
    n_q = n_k = 0;
    window(w, lane);
  }

  // Which of the row tiles from `w0` on see any key of the job.
  __device__ __forceinline__ void look(const WeighArgs& w, int lane) {
    const int tile = w0 + lane;
    Range g{0, 0, 0, 0};
    if (tile < qb) g = range_of(w, x, w.head_parts == 1 ? tile : tile / w.head_parts);
    seen = __ballot_sync(kFull, g.any_lo < k0 + KEYS && g.any_hi > k0 && g.any_lo < g.any_hi);
  }

  // Moves `w0` to the first window from there on with a row tile that sees a key of the job, or to qb.
  __device__ __forceinline__ void find(const WeighArgs& w, int lane) {
    while (w0 < qb) {
      look(w, lane);
      if (seen) return;
      w0 += 32;
    }
    w0 = qb;
    seen = 0;
  }

  // Moves to the next job; false when there is none.
  __device__ __forceinline__ bool next_job(const WeighArgs& w, int lane) {
    if (!started) {
      started = true;
      in_run = 0;
      job = static_cast<long long>(blockIdx.x) * w.run;
    } else if (++in_run < w.run) {  // the next head of the same keys
      ++job;
      ++h;
      w0 = part * w.per_part;
      seen = 1;
      if (!FEW) find(w, lane);
      return true;
    } else {
      in_run = 0;
      job += 1 + static_cast<long long>(gridDim.x - 1) * w.run;
    }
    while (job - before >= total) {
      before += total;
      r0 += 32;
      if (r0 >= w.a.R) return false;
      window(w, lane);
      x_end = 0;
    }
    const long long here = job - before;
    if (here >= x_end || here < x_begin) {  // another request
      const int src = __popc(__ballot_sync(kFull, end <= here));
      x_end = __shfl_sync(kFull, end, src);
      x_begin = src ? __shfl_sync(kFull, end, src - 1) : 0;
      x.t.r = r0 + src;
      x.t.row0 = x.t.rows = 0;
      x.t.t0 = __shfl_sync(kFull, mine.t.t0, src);
      x.t.n = __shfl_sync(kFull, mine.t.n, src);
      x.t.len = __shfl_sync(kFull, mine.t.len, src);
      x.n = __shfl_sync(kFull, mine.n, src);
      x.tiles = __shfl_sync(kFull, mine.tiles, src);
      block0 = __shfl_sync(kFull, base, src);
      if (FEW) keys = make_int2(__shfl_sync(kFull, seen_keys.x, src), __shfl_sync(kFull, seen_keys.y, src));
      if (FEW || w.parts == 1) {
        part_first = __shfl_sync(kFull, whole.x, src);
      } else {
        int2 tiles = make_int2(0, 0);
        if (lane < parts_of(w, x)) tiles = part_tiles<KEYS>(w, x, lane);
        part_first = tiles.x;
        part_end = tiles.y;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(kFull, part_end, o);
          if (lane >= o) part_end += y;
        }
      }
    }
    const unsigned within = static_cast<unsigned>(here - x_begin), hkv = w.a.L.hkv;  // (part, key tile, head)
    const int at = static_cast<int>(within / hkv);
    h = static_cast<int>(within - at * hkv);
    if (FEW || w.parts == 1) {
      part = 0;
      k0 = (part_first + at) * KEYS;
    } else {
      part = __popc(__ballot_sync(kFull, part_end <= at));
      k0 = (__shfl_sync(kFull, part_first, part) + at - (part ? __shfl_sync(kFull, part_end, part - 1) : 0)) * KEYS;
    }
    w0 = part * w.per_part;
    qb = min(x.tiles, w0 + w.per_part);
    seen = 1;
    if (FEW) return true;
    keys = part_keys(w, x, part);
    find(w, lane);
    return true;
  }

  // The next batch: of the current job, or the first of a next one.
  __device__ __forceinline__ void next(const WeighArgs& w, int lane, Batch& it) {
    it.stop = it.first = 0;
    if (!started || w0 >= qb) {
      do {
        if (!next_job(w, lane)) {
          it.stop = 1;
          return;
        }
      } while (seen == 0 && w.partial == nullptr);
      it.first = 1;
      if (seen) ++n_k;
    }
    it.h = h;
    it.k0 = k0;
    it.part = part;
    it.room = min(KEYS, x.t.len - k0);
    it.mask = seen;
    it.block0 = block0;
    it.t0 = x.t.t0;
    it.n_all = x.t.n;
    it.len = x.t.len;
    it.n = x.n;
    it.tile = w0;
    it.keys_lo = keys.x;
    it.keys_hi = keys.y;
    it.q = n_q;
    it.k = n_k - 1;
    n_q += __popc(seen);
    if (FEW) {
      w0 = qb;
    } else {
      w0 += 32;
      find(w, lane);
    }
    it.last = w0 >= qb;
  }
};

// tanh for capped scores. A score's error is the weight's relative error, and
// weights are FP32: attention's shorter polynomials (4e-7, for 16-bit outputs)
// would add up to 2e-5 of a weight under a cap of 50 to what the log-sum-exps
// carry of theirs. Odd polynomials (fitted for
// the least relative error: 2.5e-9 up to 0.25, 4.2e-9 up to 1), 1 - 2 / (1 + e^2x) beyond, whose
// absolute error of about 2^-23 is a rounding of the result there.
__device__ constexpr float kTanh4[4] = {0.999999998f, -0.333332066f, 0.133231367f, -0.0513280764f};
__device__ constexpr float kTanh8[8] = {0.999999996f,  -0.333332787f,  0.133321604f,  -0.0538709451f,
                                        0.0214648987f, -0.00791754669f, 0.00228229726f, -0.000353363486f};

template <int N>
__device__ __forceinline__ float2 cap_poly(float2 x, float cap2, const float (&c)[N]) {
  const float2 y = mul2(x, x);
  float2 p = both(cap2 * c[N - 1]);
#pragma unroll
  for (int i = N - 2; i >= 0; --i) p = fma2(p, y, both(cap2 * c[i]));
  return mul2(x, p);
}

__device__ __forceinline__ void cap_scores(float2 (&s)[kRun / 2], float c1, float cap2) {
  float far[2] = {0.f, 0.f};
#pragma unroll
  for (int j = 0; j < kRun / 2; ++j) {
    s[j] = mul2(s[j], both(c1));
    far[j & 1] = fmaxf(fmaxf(far[j & 1], fabsf(s[j].x)), fabsf(s[j].y));
  }
  const float most = fmaxf(far[0], far[1]);
  if (__all_sync(kFull, most <= 0.25f)) {
#pragma unroll
    for (int j = 0; j < kRun / 2; ++j) s[j] = cap_poly(s[j], cap2, kTanh4);
  } else {
    const bool near = __all_sync(kFull, most <= 1.f);
#pragma unroll
    for (int j = 0; j < kRun / 2; ++j) {
      const float2 x = s[j];
      s[j] = cap_poly(x, cap2, kTanh8);
      if (!near) {
        s[j].x = fabsf(x.x) <= 1.f ? s[j].x : cap2 * cap_tanh(x.x);
        s[j].y = fabsf(x.y) <= 1.f ? s[j].y : cap2 * cap_tanh(x.y);
      }
    }
  }
}

// MODE: 1 capped scores, 2 biased by distance, 3 both. RAGGED: a tile's rows do not fill the MMA's, which takes them by
// sixteens. The rows that fill it up are zeros, whose product with an infinite key is NaN: they must not be added.
// (In one kernel for both, the second form of the sums costs tiles without such rows 4 to 6 %.)
template <typename T, int D, int MODE, bool FEW, bool RAGGED>
__global__ void __launch_bounds__(Plan<D, FEW>::kThreads, 1)
weigh_tensor_kernel(const WeighArgs w, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap qmap) {
  using P = Plan<D, FEW>;
  constexpr int kSumWarps = P::kSumWarps, kThreads = P::kThreads, kInfos = P::kInfos, kBuffers = P::kBuffers;
  const PagedAttnArgs& a = w.a;
  constexpr int kHalves = D / 64;
  extern __shared__ __align__(1024) unsigned char base[];
  Shared<D, FEW>& sh = *reinterpret_cast<Shared<D, FEW>*>(base);
  const int tid = threadIdx.x, lane = tid & 31, warp = uniform(tid >> 5);
  if (warp == kSumWarps) {
    tmem_alloc(&sh.tmem, P::kTmem);
  } else if (warp == 0 && lane == 0) {
    for (int i = 0; i < P::kKRing; ++i) {
      mbar_init(&sh.k_full[i], 1);
      mbar_init(&sh.k_empty[i], 1);
    }
    for (int i = 0; i < P::kQRing; ++i) {
      mbar_init(&sh.q_full[i], 1);
      mbar_init(&sh.q_empty[i], 1);
    }
    for (int i = 0; i < kInfos; ++i) {
      mbar_init(&sh.i_full[i], 1);
      mbar_init(&sh.i_empty[i], kSumWarps + 1);
      mbar_init(&sh.i_other[i], 4 * P::kTiles);
    }
    for (int i = 0; i < P::kAhead; ++i) {
      mbar_init(&sh.w_full[i], 1);
      mbar_init(&sh.w_empty[i], kInfoWarps + kCopyWarps);
    }
    for (int i = 0; i < kBuffers; ++i) {
      mbar_init(&sh.s_full[i][0], 1);
      mbar_init(&sh.s_full[i][1], 1);
      mbar_init(&sh.s_empty[i][0], 4);
      mbar_init(&sh.s_empty[i][1], 4);
    }
    mbar_init(&sh.drained, 1);
    for (int i = 0; i < kCopyWarps; ++i) sh.k_asked[i] = sh.q_asked[i] = 0;
    fence_barrier_init();
  }
  {
    const int first = w.tokens * w.heads, n = (w.cols - first) * 8 * kHalves;  // rows that no copy writes
    for (int i = tid; i < n * P::kQRing; i += kThreads) {
      const int x = i % n, half = x % kHalves, row = first + x / (8 * kHalves);
      *reinterpret_cast<uint4*>(sh.q[i / n] + half * P::kQHalf + row * 128 + x / kHalves % 8 * 16) = make_uint4(0, 0, 0, 0);
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = uniform(sh.tmem);
  bool ok = true;

  // Batch n of the walk, for a warp that works ahead of the products.
  auto read = [&](int n, Batch& it) {
    const int slot = n % P::kAhead;
    if (!warp_wait(&sh.w_full[slot], (n / P::kAhead) & 1, a.status)) return false;
    it = sh.ahead[slot];
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.w_empty[slot]);
    return true;
  };
  if (warp > kSumWarps + 1 + kCopyWarps) {
    // ------------------------------------------------------------ rows
    const int turn = warp - kSumWarps - 2 - kCopyWarps;
    constexpr int kPasses = (P::kRows + 31) / 32;
    const int used = w.tokens * w.heads;
    int row_tok[kPasses], row_head[kPasses];
#pragma unroll
    for (int j = 0; j < kPasses; ++j) {
      row_tok[j] = (j * 32 + lane) / w.heads;
      row_head[j] = j * 32 + lane - row_tok[j] * w.heads;
    }
    int item = 0;  // all items before
    for (int n = 0; ok; ++n) {
      Batch it;
      ok = read(n, it);
      if (!ok) break;
      const bool none = it.stop || it.mask == 0;
      unsigned mask = none ? 1u : it.mask;
      bool first = it.first != 0;
      while (mask) {
        const int tile = it.tile + __ffs(mask) - 1;
        mask &= mask - 1;
        const bool now_first = first;
        first = false;
        if (item++ % kInfoWarps != turn) continue;
        const int slot = (item - 1) % kInfos;
        auto& info = sh.info[slot];
        float lse[kPasses], slope[kPasses];
        RowKeys rk[kPasses];
        bool have[kPasses];
        if (!none) {
          const int c = w.head_parts == 1 ? tile : tile / w.head_parts;
          const int at = c * w.tokens, g0 = (tile - c * w.head_parts) * w.heads;
          RowTile t;
          t.r = t.row0 = t.rows = 0;
          t.t0 = it.t0;
          t.n = it.n_all;
          t.len = it.len;
#pragma unroll
          for (int j = 0; j < kPasses; ++j) {
            const int tok = at + row_tok[j], g = g0 + row_head[j];
            have[j] = j * 32 + lane < used && tok < it.n && g < a.G;
            lse[j] = slope[j] = 0.f;
            rk[j] = RowKeys{0, 0, 0};
            if (have[j]) {
              lse[j] = w.lse[static_cast<long long>(it.t0 + tok) * a.hq + it.h * a.G + g];
              if (MODE & 2) slope[j] = a.slopes[it.h * a.G + g];
              rk[j] = row_keys(a, t, tok);
            }
          }
        }
        if (item > kInfos) ok = warp_wait(&sh.i_empty[slot], ((item - 1) / kInfos - 1) & 1, a.status);
        if (!ok) break;
        Range g{0x7fffffff, 0, 0, 0x7fffffff};
        if (!none) {
          // A row without weight (its log-sum-exp is -inf), or not there, sees no key.
#pragma unroll
          for (int j = 0; j < kPasses; ++j) {
            const int row = j * 32 + lane;
            const bool live = have[j] && lse[j] != neg_inf(), fill = row >= used;
            const int2 keys = live ? make_int2(rk[j].lo, rk[j].hi) : make_int2(0, 0);
            if (!fill) {
              g.all_lo = max(g.all_lo, keys.x);
              g.all_hi = min(g.all_hi, keys.y);
            }
            if (keys.x < keys.y) {
              g.any_lo = min(g.any_lo, keys.x);
              g.any_hi = max(g.any_hi, keys.y);
            }
            if (row < P::kRows) {
              info.neg_lse[row] = live ? -lse[j] * kLog2e : fill ? neg_inf() : 0.f;
              info.keys[row] = keys;
              if (MODE & 2) info.bias[row] = make_float2(slope[j] * kLog2e, static_cast<float>(rk[j].pos));
            }
          }
          g.any_lo = __reduce_min_sync(kFull, g.any_lo);
          g.any_hi = __reduce_max_sync(kFull, g.any_hi);
          g.all_lo = __reduce_max_sync(kFull, g.all_lo);
          g.all_hi = __reduce_min_sync(kFull, g.all_hi);
        }
        if (lane == 0) {
          Item x;
          x.h = it.h;
          x.k0 = it.k0;
          x.part = it.part;
          x.room = it.room;
          x.block0 = it.block0;
          x.first = now_first;
          x.last = it.last && mask == 0;
          x.empty = none;
          x.stop = it.stop;
          x.range = g;
          info.item = x;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.i_full[slot]);
      }
      if (it.stop) break;
    }
  } else if (warp == kSumWarps + 1 + kCopyWarps) {
    // ------------------------------------------------------------ the walk
    Walk<P::kKeys, FEW> walk;
    walk.start(w, lane);
    Batch it;
    for (int n = 0;; ++n) {
      walk.next(w, lane, it);
      const int slot = n % P::kAhead;
      if (n >= P::kAhead) ok = warp_wait(&sh.w_empty[slot], (n / P::kAhead - 1) & 1, a.status);
      if (!ok) break;
      if (lane == 0) sh.ahead[slot] = it;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.w_full[slot]);
      if (it.stop) break;
    }
  } else if (warp > kSumWarps) {
    // ------------------------------------------------------------ copies
    const int turn = warp - kSumWarps - 1;
    const bool copies_k = FEW || turn == 0, copies_q = FEW || turn == 1;
    const unsigned ps = a.L.page_size;
    const int bp = min(a.L.page_size, 128), boxes = P::kKeys / bp, ppb = a.L.b / a.L.page_size;
    const uint32_t q_bytes = static_cast<uint32_t>(w.tokens) * w.heads * D * 2;
    for (int n = 0; ok; ++n) {
      Batch it;
      ok = read(n, it);
      if (!ok || it.stop) break;
      if (it.mask == 0 || (FEW && it.q % kCopyWarps != turn)) continue;
      if (copies_k && it.first) {
        const unsigned key = it.k0 + lane * bp;
        int page = a.pages, y = static_cast<int>(key % ps / 8);
        const bool named = lane < boxes && static_cast<int>(key) < it.keys_hi && static_cast<int>(key) + bp > it.keys_lo;
        if (named)
          page = a.L.page_table[static_cast<long long>(it.block0) * ppb + key / ps];
        const int ks = it.k % P::kKRing;
        if (it.k >= P::kKRing) ok = warp_wait(&sh.k_empty[ks], (it.k / P::kKRing - 1) & 1, a.status);
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&sh.k_full[ks], P::kKBytes);
        __syncwarp();
        if (named && (page < 0 || page >= a.pages)) {  // reads as zeros
          report(a.status, kStatusBadBlockId);
          page = a.pages;
        }
        const uint32_t dst = uniform(smem_u32(sh.k[ks])), bar = uniform(smem_u32(&sh.k_full[ks]));
        for (int x = 0; x < boxes; ++x)
          tma_keys(&kmap, dst + x * bp * (D * 2), bar, __shfl_sync(kFull, y, x), __shfl_sync(kFull, page, x) * a.L.hkv + uniform(it.h));
        sh.k_asked[FEW ? turn : 0] = it.k + 1;
      }
      if (copies_q) {
        int q = it.q;
        for (unsigned mask = it.mask; mask; mask &= mask - 1, ++q) {
          const int tile = it.tile + __ffs(mask) - 1, qs = q % P::kQRing;
          if (q >= P::kQRing) ok = warp_wait(&sh.q_empty[qs], (q / P::kQRing - 1) & 1, a.status);
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(&sh.q_full[qs], q_bytes);
          __syncwarp();
          const uint32_t dst = uniform(smem_u32(sh.q[qs])), bar = uniform(smem_u32(&sh.q_full[qs]));
          const int c = w.head_parts == 1 ? tile : tile / w.head_parts;
          const int head = uniform(it.h * a.G + (tile - c * w.head_parts) * w.heads), token = uniform(it.t0 + c * w.tokens);
#pragma unroll
          for (int half = 0; half < kHalves; ++half) tma_rows(&qmap, dst + half * P::kQHalf, bar, half * 64, head, token);
          sh.q_asked[FEW ? turn : 0] = q + 1;
        }
      }
    }
  } else if (warp == kSumWarps) {
    // ------------------------------------------------------------ MMAs
    const uint32_t idesc = mma_desc<T>(128, w.cols, false);
    // K: groups of 8 keys lie D * 16 bytes apart, their 64-dim halves 1,024.
    const uint64_t k_desc = (smem_desc(smem_u32(sh.k[0]), 16) & ~(0x3fffull << 32)) | static_cast<uint64_t>(D) << 32;
    const uint64_t q_desc = smem_desc(smem_u32(sh.q[0]), 16);
    int n_info = 0, n_q = 0, n_k = 0;
    while (true) {
      const int slot = n_info % kInfos;
      ok = warp_wait(&sh.i_full[slot], (n_info / kInfos) & 1, a.status);
      if (!ok) break;
      const auto& info = sh.info[slot];
      const int stop = uniform(info.item.stop), empty = uniform(info.item.empty);
      const int first = uniform(info.item.first), last = uniform(info.item.last);
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.i_empty[slot]);
      ++n_info;
      if (stop) break;
      if (empty) continue;
      const int ks = n_k % P::kKRing, qs = n_q % P::kQRing, buf = n_q % kBuffers;
      if (first) ok = warp_wait(&sh.k_full[ks], (n_k / P::kKRing) & 1, a.status);
      ok = ok && warp_wait(&sh.q_full[qs], (n_q / P::kQRing) & 1, a.status);
      if (!ok) break;
      const uint32_t kd = uniform(static_cast<uint32_t>(k_desc) + (ks * P::kKBytes >> 4));
      const uint32_t qd = uniform(static_cast<uint32_t>(q_desc) + (qs * P::kQBytes >> 4));
      const uint32_t to = uniform(tmem + buf * P::kBufferCols);
#pragma unroll
      for (int half = 0; half < P::kTiles; ++half) {
        if (ok && n_q >= kBuffers) ok = warp_wait(&sh.s_empty[buf][half], (n_q / kBuffers - 1) & 1, a.status);
        if (!ok) break;
        fence_after();
#pragma unroll
        for (int s = 0; s < D / 16; ++s)
          mma_halves(to + half * 128, kd + ((half * 128 * D * 2 + (s >> 2) * 1024 + (s & 3) * 32) >> 4),
                     static_cast<uint32_t>(k_desc >> 32), qd + (((s >> 2) * P::kQHalf + (s & 3) * 32) >> 4),
                     static_cast<uint32_t>(q_desc >> 32), idesc, s > 0);
        mma_commit(&sh.s_full[buf][half]);
      }
      if (!ok) break;
      mma_commit(&sh.q_empty[qs]);
      ++n_q;
      if (last) {
        mma_commit(&sh.k_empty[ks]);
        ++n_k;
      }
    }
    mma_commit(&sh.drained);  // products under way end before tensor memory is freed
    warp_wait(&sh.drained, 0, a.status);
  } else {
    // ------------------------------------------------------------ weights
    const int half = (warp >> 2) % P::kTiles, group = warp / (4 * P::kTiles);
    const int mine = half * 128 + (warp & 3) * 32;  // first of the warp's keys in the job
    const uint32_t ts = tmem + (static_cast<uint32_t>(warp & 3) << 21) + half * 128;
    const float c = (MODE & 1) ? a.scale / a.softcap : a.scale * kLog2e, cap2 = a.softcap * kLog2e;
    const int cols = w.cols, used = w.tokens * w.heads;
    float2 sum = make_float2(0.f, 0.f);
    int n_info = 0, n_s = 0;
    while (true) {
      const int slot = n_info % kInfos;
      ok = warp_wait(&sh.i_full[slot], (n_info / kInfos) & 1, a.status);
      if (!ok) break;
      auto& info = sh.info[slot];
      const Item it = info.item;
      if (it.stop) break;
      if (it.first) sum = make_float2(0.f, 0.f);
      const int first_key = it.k0 + mine, key = first_key + lane;
      // The groups take every second row tile each.
      const bool own = P::kGroups == 1 || (it.empty ? 0 : n_s & 1) == group;
      if (!it.empty && !own) {
        ++n_s;
      } else if (!it.empty) {
        const int buf = n_s % kBuffers;
        ok = warp_wait(&sh.s_full[buf][half], (n_s / kBuffers) & 1, a.status);
        if (!ok) break;
        fence_after();
        const Range g = it.range;
        const bool none = g.any_lo >= first_key + 32 || g.any_hi <= first_key;
        const bool whole = g.all_lo <= first_key && g.all_hi >= first_key + 32;
        auto release = [&]() {  // the warp has read its S
          fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.s_empty[buf][half]);
        };
        float2 part[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        auto tile = [&](auto whole_t) {
          constexpr bool WHOLE = decltype(whole_t)::value;
          float2 s[2][kRun / 2];
          tmem_ld16(ts + buf * P::kBufferCols, reinterpret_cast<uint32_t*>(s[0]));
          auto run = [&](float2 (&x)[kRun / 2], int j) {
            if (RAGGED && !FEW && WHOLE && j + kRun > used) {  // rows that fill up: scores of 0, log-sum-exps of infinity
#pragma unroll
              for (int e = 0; e < kRun / 2; ++e) {
                x[e].x = j + 2 * e < used ? x[e].x : 0.f;
                x[e].y = j + 2 * e + 1 < used ? x[e].y : 0.f;
              }
            }
            if (MODE & 1) cap_scores(x, c, cap2);
            float4 l4;
#pragma unroll
            for (int e = 0; e < kRun / 2; ++e) {
              if (RAGGED && FEW && 2 * e >= used) break;
              if (e % 2 == 0) l4 = *reinterpret_cast<const float4*>(&info.neg_lse[j + 2 * e]);
              const float2 l = e % 2 ? make_float2(l4.z, l4.w) : make_float2(l4.x, l4.y);
              float2 y;
              if (MODE & 2) {
                const float4 b = *reinterpret_cast<const float4*>(&info.bias[j + 2 * e]);
                const float at = static_cast<float>(key);
                y = (MODE & 1) ? x[e] : mul2(x[e], both(c));
                y.x = fmaf(-b.x, fabsf(b.y - at), y.x);
                y.y = fmaf(-b.z, fabsf(b.w - at), y.y);
                y = add2(y, l);
              } else {
                y = (MODE & 1) ? add2(x[e], l) : fma2(x[e], both(c), l);
              }
              y = make_float2(ex2(y.x), ex2(y.y));
              if (!WHOLE) {
                const int4 k = *reinterpret_cast<const int4*>(&info.keys[j + 2 * e]);
                y.x = key >= k.x && key < k.y ? y.x : 0.f;
                y.y = key >= k.z && key < k.w ? y.y : 0.f;
              } else if (RAGGED && FEW) {
                y.y = 2 * e + 1 < used ? y.y : 0.f;
              }
              part[e & 1] = add2(part[e & 1], y);
            }
          };
#pragma unroll 1
          for (int j = 0; j < cols; j += 2 * kRun) {
            tmem_wait_ld();
            tmem_loaded<kRun>(reinterpret_cast<uint32_t*>(s[0]));
            const bool more = j + kRun < cols;
            if (more) tmem_ld16(ts + buf * P::kBufferCols + j + kRun, reinterpret_cast<uint32_t*>(s[1]));
            else release();
            run(s[0], j);
            if (more) {
              tmem_wait_ld();
              tmem_loaded<kRun>(reinterpret_cast<uint32_t*>(s[1]));
              if (j + 2 * kRun < cols) tmem_ld16(ts + buf * P::kBufferCols + j + 2 * kRun, reinterpret_cast<uint32_t*>(s[0]));
              else release();
              run(s[1], j + kRun);
            }
          }
        };
        if (!none) {
          if (whole) tile(std::true_type{});
          else tile(std::false_type{});
        } else {
          release();
        }
        ++n_s;
        part[0] = add2(part[0], part[1]);
        sum = add2(sum, part[0]);
      }
      if (!own) {
        if (it.last) info.other[mine + lane] = sum.x + sum.y;
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.i_other[slot]);
      } else if (it.last) {
        float x = sum.x + sum.y;
        if (P::kGroups == 2) {
          ok = warp_wait(&sh.i_other[slot], (n_info / kInfos) & 1, a.status);
          if (!ok) break;
          x += info.other[mine + lane];
        }
        if (mine + lane < it.room) {
          const long long at = it.h * w.slots + static_cast<long long>(it.block0) * a.L.b + key;
          if (w.partial) w.partial[it.part * w.slots * a.L.hkv + at] = x;
          else if (x != 0.f) atomicAdd(w.weights + at, x);  // the key's only one of the call: nothing waits for it
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.i_empty[slot]);
      ++n_info;
    }
  }
  fence_before();
  __syncthreads();
  if (warp == kSumWarps) {
    fence_after();
    tmem_free(tmem, P::kTmem);
  } else if (warp == 0) {
    // After a wait that ran out the CTA does not end under copies that nobody waited for.
    for (int c = 0; c < kCopyWarps; ++c) {
      const int step = FEW ? kCopyWarps : 1;
      for (int i = sh.k_asked[c] - 1; i >= 0 && i > sh.k_asked[c] - 1 - P::kKRing; i -= step)
        if (!warp_wait(&sh.k_full[i % P::kKRing], (i / P::kKRing) & 1, a.status)) break;
      for (int i = sh.q_asked[c] - 1; i >= 0 && i > sh.q_asked[c] - 1 - P::kQRing; i -= step)
        if (!warp_wait(&sh.q_full[i % P::kQRing], (i / P::kQRing) & 1, a.status)) break;
    }
  }
}

// What each chunk of w.tokens tokens, and each part, sees, for masks that are
// given. A CTA per part.
__global__ void __launch_bounds__(256) weigh_ranges_kernel(const WeighArgs w) {
  __shared__ int2 of_warp[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r = blockIdx.x / w.parts, p = blockIdx.x % w.parts;
  const Rows x = rows_of(w, r);
  const long long at = weigh_range_at(x.t.t0, r, w.tokens);
  int lo = 0x7fffffff, hi = 0;
  for (int q = p * w.per_part + warp * w.head_parts; q < min(x.tiles, (p + 1) * w.per_part); q += 8 * w.head_parts) {
    const int c = q / w.head_parts;  // (a chunk that two parts share is written twice, alike)
    Range g{0x7fffffff, 0, 0, 0x7fffffff};
    for (int i = c * w.tokens + lane; i < min(x.n, (c + 1) * w.tokens); i += 32) {
      const RowKeys k = row_keys(w.a, x.t, i);
      g.all_lo = max(g.all_lo, k.lo);
      g.all_hi = min(g.all_hi, k.hi);
      if (k.lo < k.hi) {
        g.any_lo = min(g.any_lo, k.lo);
        g.any_hi = max(g.any_hi, k.hi);
      }
    }
    g.any_lo = __reduce_min_sync(kFull, g.any_lo);
    g.any_hi = __reduce_max_sync(kFull, g.any_hi);
    g.all_lo = __reduce_max_sync(kFull, g.all_lo);
    g.all_hi = __reduce_min_sync(kFull, g.all_hi);
    if (lane == 0) w.ranges[at + c] = make_int4(g.any_lo, g.any_hi, g.all_lo, g.all_hi);
    lo = min(lo, g.any_lo);
    hi = max(hi, g.any_hi);
  }
  if (lane == 0) of_warp[warp] = make_int2(lo, hi);
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 0; i < 8; ++i) {
      lo = min(lo, of_warp[i].x);
      hi = max(hi, of_warp[i].y);
    }
    w.part_keys[blockIdx.x] = make_int2(lo, hi);
  }
}

// weights += the parts' sums, in the order of the parts.
template <int KEYS>
__global__ void __launch_bounds__(256) weigh_join_kernel(const WeighArgs w, int tiles) {
  const int tile = static_cast<int>(blockIdx.x % tiles);
  const int h = static_cast<int>(blockIdx.x / tiles) % w.a.L.hkv, r = static_cast<int>(blockIdx.x / tiles) / w.a.L.hkv;
  const Rows x = rows_of(w, r);
  const int key = tile * 256 + threadIdx.x;
  if (x.n == 0 || key >= x.t.len) return;
  const int parts = parts_of(w, x);
  const long long at = h * w.slots + static_cast<long long>(w.a.L.block_offsets[r]) * w.a.L.b + key;
  float sum = 0.f;
  for (int p = 0; p < parts; ++p) {
    const int2 t = part_tiles<KEYS>(w, x, p);
    if (key / KEYS >= t.x && key / KEYS < t.x + t.y) sum += w.partial[p * w.slots * w.a.L.hkv + at];
  }
  if (sum != 0.f) w.weights[at] += sum;
}

// A tensor map over K of the page pool: (64 dims, 8 keys, halves of a head,
// groups of 8 keys, page and head); a box is a page of one head, or 128 keys of
// it, in one copy.
int encode_key_map(CUtensorMap* map, const PagedAttnArgs& a, int kv_dtype) {
  const EncodeTiled fn = encode_tiled();
  if (fn == nullptr) return static_cast<int>(cudaErrorNotSupported);
  const cuuint64_t d = a.d, ps = a.L.page_size, halves = d / 64;
  const cuuint64_t dims[5] = {64, 8, halves, ps / 8, static_cast<cuuint64_t>(a.pages) * a.L.hkv};
  const cuuint64_t strides[4] = {d * 2, 128, d * 16, ps * d * 2};
  const cuuint32_t box[5] = {64, 8, static_cast<cuuint32_t>(halves), static_cast<cuuint32_t>((ps < 128 ? ps : 128) / 8), 1};
  const cuuint32_t step[5] = {1, 1, 1, 1, 1};
  const CUresult r = fn(map, kv_dtype == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5,
                        const_cast<void*>(a.L.k), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : static_cast<int>(cudaErrorInvalidValue);
}

// A tensor map over the queries: boxes of 64 dims x w.heads heads x w.tokens tokens, 128-byte swizzle.
int encode_query_map(CUtensorMap* map, const WeighArgs& w, int kv_dtype) {
  const PagedAttnArgs& a = w.a;
  const EncodeTiled fn = encode_tiled();
  if (fn == nullptr) return static_cast<int>(cudaErrorNotSupported);
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(a.d), static_cast<cuuint64_t>(a.hq), static_cast<cuuint64_t>(a.T), 1};
  const cuuint64_t token = static_cast<cuuint64_t>(a.q_ts) * 2, head = static_cast<cuuint64_t>(a.q_hs) * 2;
  const cuuint64_t strides[3] = {head, token, token > head ? token : head};  // (one place along the last axis)
  const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(w.heads), static_cast<cuuint32_t>(w.tokens), 1};
  const cuuint32_t step[4] = {1, 1, 1, 1};
  const CUresult r = fn(map, kv_dtype == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                        const_cast<void*>(a.q), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : kWeighNoMap;
}

template <typename T, int D, int MODE, bool FEW, bool RAGGED>
int launch_kernel(const WeighArgs& w, int sms, const CUtensorMap& km, const CUtensorMap& qm, cudaStream_t stream) {
  constexpr int bytes = sizeof(Shared<D, FEW>);
  static_assert(bytes <= 227 * 1024, "shared memory of a CTA");
  auto kern = weigh_tensor_kernel<T, D, MODE, FEW, RAGGED>;
  const int rc = static_cast<int>(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  if (rc) return rc;
  kern<<<sms, Plan<D, FEW>::kThreads, bytes, stream>>>(w, km, qm);
  return static_cast<int>(cudaGetLastError());
}

template <typename T, int D, int MODE, bool FEW>
int launch_mode(const WeighArgs& w, int sms, const CUtensorMap& km, const CUtensorMap& qm, cudaStream_t stream) {
  if (FEW || w.tokens * w.heads < w.cols) return launch_kernel<T, D, MODE, FEW, true>(w, sms, km, qm, stream);
  return launch_kernel<T, D, MODE, FEW, FEW>(w, sms, km, qm, stream);
}

template <typename T, int D, bool FEW>
int launch_d(const WeighArgs& w, int sms, const CUtensorMap& km, const CUtensorMap& qm, cudaStream_t stream) {
  switch ((w.a.softcap > 0.f ? 1 : 0) | (w.a.slopes ? 2 : 0)) {
    case 0: return launch_mode<T, D, 0, FEW>(w, sms, km, qm, stream);
    case 1: return launch_mode<T, D, 1, FEW>(w, sms, km, qm, stream);
    case 2: return launch_mode<T, D, 2, FEW>(w, sms, km, qm, stream);
    default: return launch_mode<T, D, 3, FEW>(w, sms, km, qm, stream);
  }
}

template <typename T>
int launch_t(const WeighArgs& w, int sms, const CUtensorMap& km, const CUtensorMap& qm, cudaStream_t stream) {
  if (w.few) return w.a.d == 64 ? launch_d<T, 64, true>(w, sms, km, qm, stream) : launch_d<T, 128, true>(w, sms, km, qm, stream);
  return w.a.d == 64 ? launch_d<T, 64, false>(w, sms, km, qm, stream) : launch_d<T, 128, false>(w, sms, km, qm, stream);
}

}  // namespace

// 16-bit types, heads of 64 or 128 dims, pages that tile 128 keys (or are
// tiled by them), 16-byte rows of queries and keys.
bool weigh_tensor_takes(int kv_dtype, int d, int page_size, const void* k, const void* q, long long q_ts, long long q_hs) {
  const bool pages = page_size >= 8 && (page_size <= 128 ? 128 % page_size == 0 : page_size % 128 == 0);
  const uintptr_t any = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(q) | static_cast<uintptr_t>(q_ts * 2) |
                        static_cast<uintptr_t>(q_hs * 2);
  return kv_dtype != kF32 && (d == 64 || d == 128) && pages && any % 16 == 0 && q_ts > 0 && q_hs > 0;
}

int launch_weigh_tensor(const WeighArgs& w, int kv_dtype, int sms, cudaStream_t stream) {
  CUtensorMap km, qm;
  int rc = encode_key_map(&km, w.a, kv_dtype);
  if (rc) return rc;
  rc = encode_query_map(&qm, w, kv_dtype);
  if (rc) return rc;
  const int tiles = (w.longest + 255) / 256;
  const long long ctas = static_cast<long long>(w.a.R) * w.parts, joins = static_cast<long long>(tiles) * w.a.L.hkv * w.a.R;
  if ((w.partial && joins > 0x7fffffff) || (w.ranges && ctas > 0x7fffffff)) return static_cast<int>(cudaErrorInvalidValue);
  if (w.ranges) {
    weigh_ranges_kernel<<<static_cast<unsigned>(ctas), 256, 0, stream>>>(w);
    rc = static_cast<int>(cudaGetLastError());
    if (rc) return rc;
  }
  rc = kv_dtype == kBF16 ? launch_t<__nv_bfloat16>(w, sms, km, qm, stream) : launch_t<__half>(w, sms, km, qm, stream);
  if (rc || !w.partial) return rc;
  const auto join = w.few ? weigh_join_kernel<128> : weigh_join_kernel<256>;
  join<<<static_cast<unsigned>(joins), 256, 0, stream>>>(w, tiles);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace stk
