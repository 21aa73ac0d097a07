// Attention weight received by each cached key, on the tensor cores (tcgen05).
//
// The sum over rows (new tokens x query heads of the group) of 2^(c s - lse) is
// taken per key, so S is formed with the keys along the tensor memory's lanes:
//   S^T = K Q^T        128 keys x up to 112 rows, FP32 in tensor memory
//   sum += 2^(c S - lse)   one thread per key; a row's log-sum-exp, known
//                          beforehand, is the same for all of a warp's keys
// No running maximum, no reduction across threads, no atomics: a key's sum is
// taken in the order of its rows.
//
// A job is 256 keys of one request's KV head and a part of its rows. The CTAs of a
// persistent grid (one per SM) take every gridDim'th job; copies run ahead of
// the products across the borders of jobs, the next job's K under the current
// one's rows. With single tokens K streams through, with prompts the row tiles
// do, one in shared memory for both halves of the keys (a tile from L2 serves
// 256 x 112 scores: half of what 128 keys would ask of L2).
//
// Warps 0-7: exponentials and sums, one M tile of 128 keys each four. Warp 8:
// MMAs. Warps 9-12: the walk over jobs and row tiles, log-sum-exps and key
// intervals of the tiles' rows, K (warp 10) and Q (warp 9) by TMA.
//
// Rows that see none of a warp's keys are skipped tile by tile, tiles whose
// rows all see all of a warp's keys need no mask. Unseen keys may hold
// anything: each key is a lane of its own, selected, never multiplied. Boxes
// of keys that no row of the job sees are not looked up and read as zeros.

#include "paged_tensor.cuh"
#include "tcgen05.cuh"
#include "weigh.cuh"

namespace stk {

int set_wait_limit_weigh(unsigned long long ns) { return set_wait_limit_this_unit(ns); }

namespace {

constexpr int kSumWarps = 8, kLoadWarps = 4, kThreads = (kSumWarps + 1 + kLoadWarps) * 32;
constexpr int kBuffers = 2;  // S tiles in tensor memory, each 2 x 128 columns
constexpr int kInfos = 4;    // row tiles whose rows' data are held
constexpr int kRun = 16;     // rows taken from tensor memory at once

// Keys that a row tile's rows see: least and largest of any, and of all.
struct Range {
  int any_lo, any_hi, all_lo, all_hi;
};

struct Item {
  int r, h, k0, part;  // job: request, KV head, first key, part
  int first, last;     // of the job
  int empty;           // a job without rows: only its zeros are to be written
  int stop;
  int cols;
  Range range;
  long long slot;      // of the request's first key, among the head's
  int room;            // keys from k0 on that have slots
};

struct Info {
  Item item;
  int odd[kLoadWarps];                      // a warp's rows are not all there, or have no weight
  alignas(16) float neg_lse[kWeighRows];    // - log-sum-exp * log2 e
  alignas(16) float2 bias[kWeighRows];      // slope * log2 e, place
  alignas(16) int2 keys[kWeighRows];        // lo, hi
};

template <int D>
struct Plan {
  static constexpr int kKBytes = kWeighKeys * D * 2, kKHalf = kWeighKeys * 128;
  static constexpr int kQBytes = kWeighRows * D * 2, kQHalf = kWeighRows * 128;
  static constexpr int kKRing = 2, kQRing = D == 128 ? 3 : 6;
};

template <int D>
struct Shared {
  alignas(1024) unsigned char k[Plan<D>::kKRing][Plan<D>::kKBytes];
  alignas(1024) unsigned char q[Plan<D>::kQRing][Plan<D>::kQBytes];
  Info info[kInfos];
  uint64_t k_full[Plan<D>::kKRing], k_empty[Plan<D>::kKRing];
  uint64_t q_full[Plan<D>::kQRing], q_empty[Plan<D>::kQRing];
  uint64_t i_full[kInfos], i_empty[kInfos];
  uint64_t s_full[kBuffers][2], s_empty[kBuffers];
  uint64_t drained;
  volatile int k_asked, q_asked;  // copies asked for
  uint32_t tmem;
};

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

// Keys that tokens [i, i + w.tokens) of a request see under the causal mask.
__device__ __forceinline__ Range causal_range(const WeighArgs& w, const Rows& x, int i) {
  const int pos = x.t.len - x.t.n + i, last = min(w.tokens, x.n - i) - 1;
  Range g;
  g.any_lo = g.all_lo = 0;
  g.any_hi = max(0, min(pos + last + 1, x.t.len));
  g.all_hi = max(0, min(pos + 1, x.t.len));
  return g;
}

// A warp's walk over the CTA's jobs and their row tiles. Four warps walk alike.
struct Walk {
  // a window of 32 requests, one per lane
  int r0;
  Rows mine;
  int key_tiles;
  long long end, total, before;  // jobs up to the lane's request, of the window, before the window
  long long job;
  // the current job
  Rows x;
  int h, k0, part, first_row;
  long long slot;
  int room;
  int q, qb;             // next row tile, end of the job's
  // a window of 32 row tiles from `w0` on
  int w0;
  Range range;
  unsigned seen;
  bool started;

  __device__ __forceinline__ void window(const WeighArgs& w, int lane) {
    const int r = r0 + lane;
    mine = Rows{};
    key_tiles = 0;
    long long jobs = 0;
    if (r < w.a.R) {
      mine = rows_of(w, r);
      key_tiles = mine.n > 0 ? (mine.t.len + kWeighKeys - 1) / kWeighKeys : 0;
      const int parts = (mine.tiles + w.per_part - 1) / w.per_part;
      jobs = static_cast<long long>(key_tiles) * parts * w.a.L.hkv;
    }
    end = jobs;
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
    job = static_cast<long long>(blockIdx.x) - gridDim.x;
    started = false;
    window(w, lane);
  }

  // The row tiles from `w0` on: what they see, and which see any key of the job.
  __device__ __forceinline__ void look(const WeighArgs& w, int lane) {
    const int tile = w0 + lane;
    range = Range{0x7fffffff, 0, 0x7fffffff, 0};
    if (tile < qb) {
      const int c = tile / w.head_parts;
      if (w.ranges) {
        const int4 g = w.ranges[weigh_range_at(x.t.t0, x.t.r, w.tokens) + c];
        range = Range{g.x, g.y, g.z, g.w};
      } else {
        range = causal_range(w, x, c * w.tokens);
      }
    }
    seen = __ballot_sync(kFull, tile < qb && range.any_lo < k0 + kWeighKeys && range.any_hi > k0 && range.any_lo < range.any_hi);
  }

  // The first row tile from q on that sees a key of the job: q, or qb if there is none.
  __device__ __forceinline__ void find(const WeighArgs& w, int lane) {
    while (q < qb) {
      if (q >= w0 + 32) {
        w0 = q;
        look(w, lane);
      }
      const unsigned m = seen >> (q - w0) << (q - w0);
      if (m) {
        q = w0 + __ffs(m) - 1;
        return;
      }
      q = w0 + 32;
    }
    q = qb;
  }

  // Moves to the next job; false when there is none.
  __device__ __forceinline__ bool next_job(const WeighArgs& w, int lane) {
    job += gridDim.x;
    while (job - before >= total) {
      before += total;
      r0 += 32;
      if (r0 >= w.a.R) return false;
      window(w, lane);
    }
    const int src = __popc(__ballot_sync(kFull, end <= job - before));
    const long long begin = src ? __shfl_sync(kFull, end, src - 1) : 0;
    x.t.r = r0 + src;
    x.t.row0 = x.t.rows = 0;
    x.t.t0 = __shfl_sync(kFull, mine.t.t0, src);
    x.t.n = __shfl_sync(kFull, mine.t.n, src);
    x.t.len = __shfl_sync(kFull, mine.t.len, src);
    x.n = __shfl_sync(kFull, mine.n, src);
    x.tiles = __shfl_sync(kFull, mine.tiles, src);
    const int tiles = __shfl_sync(kFull, key_tiles, src);
    int at = static_cast<int>(job - before - begin);  // (part, key tile, head)
    h = at % w.a.L.hkv;
    at /= w.a.L.hkv;
    k0 = at % tiles * kWeighKeys;
    part = at / tiles;
    slot = static_cast<long long>(w.a.L.block_offsets[x.t.r]) * w.a.L.b;
    room = min(kWeighKeys, x.t.len - k0);
    q = part * w.per_part;
    qb = min(x.tiles, q + w.per_part);
    w0 = q;
    look(w, lane);
    find(w, lane);
    return true;
  }

  // The next item: a row tile of the current job, or the first of a next one.
  __device__ __forceinline__ void next(const WeighArgs& w, int lane, Item& it) {
    it.stop = it.empty = it.first = 0;
    if (!started || q >= qb) {
      do {
        started = true;
        if (!next_job(w, lane)) {
          it.stop = 1;
          return;
        }
      } while (q >= qb && w.partial == nullptr);
      it.first = 1;
      it.empty = q >= qb;
    }
    it.r = x.t.r;
    it.h = h;
    it.k0 = k0;
    it.part = part;
    it.slot = slot;
    it.room = room;
    it.cols = w.cols;
    it.last = 1;
    first_row = q;
    if (it.empty) return;
    const int src = q - w0;
    it.range.any_lo = __shfl_sync(kFull, range.any_lo, src);
    it.range.any_hi = __shfl_sync(kFull, range.any_hi, src);
    it.range.all_lo = __shfl_sync(kFull, range.all_lo, src);
    it.range.all_hi = __shfl_sync(kFull, range.all_hi, src);
    ++q;
    find(w, lane);
    it.last = q >= qb;
  }

  // The keys [.x, .y) that any of the job's rows sees; the row tiles' window is the first one's.
  __device__ __forceinline__ int2 job_keys(const WeighArgs& w, int lane) {
    if (w.ranges == nullptr) return make_int2(0, x.t.len);
    int lo = 0x7fffffff, hi = 0;
    for (int c = part * w.per_part / w.head_parts + lane; c * w.head_parts < qb; c += 32) {
      const int4 g = w.ranges[weigh_range_at(x.t.t0, x.t.r, w.tokens) + c];
      if (g.x < g.y) {
        lo = min(lo, g.x);
        hi = max(hi, g.y);
      }
    }
    return make_int2(__reduce_min_sync(kFull, lo), __reduce_max_sync(kFull, hi));
  }
};

// tanh for capped scores: odd polynomials in the raw score (least relative
// error, fitted: 2.5e-9 up to 0.25, 4.2e-9 up to 1), the function beyond.
__device__ constexpr float kTanh4[4] = {0.999999998f, -0.333332066f, 0.133231367f, -0.0513280764f};
__device__ constexpr float kTanh8[8] = {0.999999996f,  -0.333332787f,  0.133321604f,  -0.0538709451f,
                                        0.0214648987f, -0.00791754669f, 0.00228229726f, -0.000353363486f};

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
    for (int j = 0; j < kRun / 2; ++j) {
      const float2 y = mul2(s[j], s[j]);
      float2 p = both(cap2 * kTanh4[3]);
#pragma unroll
      for (int i = 2; i >= 0; --i) p = fma2(p, y, both(cap2 * kTanh4[i]));
      s[j] = mul2(s[j], p);
    }
  } else if (__all_sync(kFull, most <= 1.f)) {
#pragma unroll
    for (int j = 0; j < kRun / 2; ++j) {
      const float2 y = mul2(s[j], s[j]);
      float2 p = both(cap2 * kTanh8[7]);
#pragma unroll
      for (int i = 6; i >= 0; --i) p = fma2(p, y, both(cap2 * kTanh8[i]));
      s[j] = mul2(s[j], p);
    }
  } else {
#pragma unroll 1
    for (int j = 0; j < kRun / 2; ++j) s[j] = make_float2(cap2 * tanhf(s[j].x), cap2 * tanhf(s[j].y));
  }
}

// MODE: 1 capped scores, 2 biased by distance, 3 both.
template <typename T, int D, int MODE>
__global__ void __launch_bounds__(kThreads, 1)
weigh_tensor_kernel(const WeighArgs w, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap qmap) {
  using P = Plan<D>;
  const PagedAttnArgs& a = w.a;
  constexpr int kHalves = D / 64;
  extern __shared__ __align__(1024) unsigned char base[];
  Shared<D>& sh = *reinterpret_cast<Shared<D>*>(base);
  const int tid = threadIdx.x, lane = tid & 31, warp = uniform(tid >> 5);
  if (warp == kSumWarps) {
    tmem_alloc(&sh.tmem, 512);
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
      mbar_init(&sh.i_full[i], kLoadWarps);
      mbar_init(&sh.i_empty[i], kSumWarps + 1);
    }
    for (int i = 0; i < kBuffers; ++i) {
      mbar_init(&sh.s_full[i][0], 1);
      mbar_init(&sh.s_full[i][1], 1);
      mbar_init(&sh.s_empty[i], kSumWarps);
    }
    mbar_init(&sh.drained, 1);
    sh.k_asked = sh.q_asked = 0;
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

  if (warp > kSumWarps) {
    // ------------------------------------------------------------ jobs, rows, copies
    const int lw = warp - kSumWarps - 1, row = lw * 32 + lane;
    const int row_tok = row / w.heads, row_head = row - row_tok * w.heads;
    const int bp = min(a.L.page_size, 128), boxes = kWeighKeys / bp;
    const uint32_t q_bytes = static_cast<uint32_t>(w.tokens) * w.heads * D * 2;
    Walk walk;
    walk.start(w, lane);
    Item now, then;
    struct Mine {
      float lse, slope;
      RowKeys rk;
      bool have;
      int page, kq;  // K boxes of a job's first tile; row tile
    };
    // Loads of the lane's row (and, warp 1, its box of K) of an item: under way while the item before is handed on.
    auto fetch = [&](const Item& it) {
      Mine m{};
      if (it.stop || it.empty) return m;
      m.kq = walk.first_row;
      const int c = m.kq / w.head_parts, tok = c * w.tokens + row_tok;
      const int g = (m.kq - c * w.head_parts) * w.heads + row_head;
      m.have = row < w.tokens * w.heads && tok < walk.x.n && g < a.G;
      if (m.have) {
        m.lse = w.lse[static_cast<long long>(walk.x.t.t0 + tok) * a.hq + it.h * a.G + g];
        m.slope = (MODE & 2) ? a.slopes[it.h * a.G + g] : 0.f;
        m.rk = row_keys(a, walk.x.t, tok);
      }
      if (lw == 1 && it.first) {
        const int2 keys = walk.job_keys(w, lane);
        const int key = it.k0 + lane * bp;
        m.page = a.pages;
        if (lane < boxes && key < keys.y && key + bp > keys.x) {
          const int page = page_of(a, it.r, key);
          m.page = page < 0 ? a.pages : page;
        }
      }
      return m;
    };
    int n_info = 0, n_q = 0, n_k = 0;
    walk.next(w, lane, now);
    int t0 = walk.x.t.t0;
    Mine m = fetch(now);
    while (true) {
      then.stop = 1;
      int t0_then = 0;
      Mine mt{};
      if (!now.stop) {
        walk.next(w, lane, then);
        t0_then = walk.x.t.t0;
        mt = fetch(then);
      }
      const int slot = n_info % kInfos;
      if (n_info >= kInfos) ok = warp_wait(&sh.i_empty[slot], (n_info / kInfos - 1) & 1, a.status);
      if (!ok) break;
      Info& info = sh.info[slot];
      if (lw == 0 && lane == 0) info.item = now;
      if (!now.stop && !now.empty) {
        // A row without weight (its log-sum-exp is -inf) sees no key. Rows that only fill up the MMA's are zeros
        // with a log-sum-exp of infinity.
        const bool live = m.have && m.lse != neg_inf(), fill = row >= w.tokens * w.heads;
        if (row < kWeighRows) {
          info.neg_lse[row] = live ? -m.lse * kLog2e : fill ? neg_inf() : 0.f;
          info.keys[row] = live ? make_int2(m.rk.lo, m.rk.hi) : make_int2(0, 0);
          if (MODE & 2) info.bias[row] = make_float2(m.slope * kLog2e, static_cast<float>(m.rk.pos));
        }
        const bool odd = __any_sync(kFull, !fill && !live);
        if (lane == 0) info.odd[lw] = odd;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.i_full[slot]);
      ++n_info;
      if (now.stop) break;
      if (!now.empty) {
        if (lw == 1 && now.first) {
          const int ks = n_k % P::kKRing;
          if (n_k >= P::kKRing) ok = warp_wait(&sh.k_empty[ks], (n_k / P::kKRing - 1) & 1, a.status);
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(&sh.k_full[ks], P::kKBytes);
          __syncwarp();
          if (lane < boxes) {
            const int y = (now.k0 + lane * bp) % a.L.page_size;
#pragma unroll
            for (int half = 0; half < kHalves; ++half)
              tma_load(&kmap, sh.k[ks] + half * P::kKHalf + lane * bp * 128, &sh.k_full[ks], half * 64, y, now.h, m.page);
          }
          __syncwarp();
          sh.k_asked = ++n_k;
        }
        if (lw == 0) {
          const int qs = n_q % P::kQRing;
          if (n_q >= P::kQRing) ok = warp_wait(&sh.q_empty[qs], (n_q / P::kQRing - 1) & 1, a.status);
          if (!ok) break;
          if (lane == 0) {
            mbar_arrive_expect_tx(&sh.q_full[qs], q_bytes);
            const int c = m.kq / w.head_parts;
#pragma unroll
            for (int half = 0; half < kHalves; ++half)
              tma_load(&qmap, sh.q[qs] + half * P::kQHalf, &sh.q_full[qs], half * 64,
                       now.h * a.G + (m.kq - c * w.head_parts) * w.heads, t0 + c * w.tokens, 0);
          }
          __syncwarp();
          sh.q_asked = ++n_q;
        }
      }
      now = then;
      m = mt;
      t0 = t0_then;
    }
  } else if (warp == kSumWarps) {
    // ------------------------------------------------------------ MMAs
    const uint32_t idesc = mma_desc<T>(128, w.cols, false);
    const uint64_t k_desc = smem_desc(smem_u32(sh.k[0]), 16), q_desc = smem_desc(smem_u32(sh.q[0]), 16);
    int n_info = 0, n_q = 0, n_k = 0;
    while (true) {
      const int slot = n_info % kInfos;
      ok = warp_wait(&sh.i_full[slot], (n_info / kInfos) & 1, a.status);
      if (!ok) break;
      const Info& info = sh.info[slot];
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
      if (ok && n_q >= kBuffers) ok = warp_wait(&sh.s_empty[buf], (n_q / kBuffers - 1) & 1, a.status);
      if (!ok) break;
      fence_after();
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint64_t kd = k_desc + ((ks * P::kKBytes + half * 128 * 128) >> 4), qd = q_desc + (qs * P::kQBytes >> 4);
#pragma unroll
        for (int s = 0; s < D / 16; ++s)
          mma_ss(tmem + (buf * 2 + half) * 128, kd + (((s >> 2) * P::kKHalf + (s & 3) * 32) >> 4),
                 qd + (((s >> 2) * P::kQHalf + (s & 3) * 32) >> 4), idesc, s > 0);
        mma_commit(&sh.s_full[buf][half]);
      }
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
    const int half = warp >> 2, mine = half * 128 + (warp & 3) * 32;  // first of the warp's keys in the job
    const uint32_t ts = tmem + (static_cast<uint32_t>(warp & 3) << 21) + half * 128;
    const float c = (MODE & 1) ? a.scale / a.softcap : a.scale * kLog2e, cap2 = a.softcap * kLog2e;
    float2 sum = make_float2(0.f, 0.f);
    int n_info = 0, n_s = 0;
    while (true) {
      const int slot = n_info % kInfos;
      ok = warp_wait(&sh.i_full[slot], (n_info / kInfos) & 1, a.status);
      if (!ok) break;
      const Info& info = sh.info[slot];
      if (uniform(info.item.stop)) break;
      if (uniform(info.item.first)) sum = make_float2(0.f, 0.f);
      const int first_key = uniform(info.item.k0) + mine, key = first_key + lane;
      if (!uniform(info.item.empty)) {
        const int buf = n_s % kBuffers, cols = uniform(info.item.cols);
        ok = warp_wait(&sh.s_full[buf][half], (n_s / kBuffers) & 1, a.status);
        if (!ok) break;
        fence_after();
        const Range g = info.item.range;
        const bool none = g.any_lo >= first_key + 32 || g.any_hi <= first_key;
        const bool odd = (info.odd[0] | info.odd[1] | info.odd[2] | info.odd[3]) != 0;
        const bool whole = !odd && g.all_lo <= first_key && g.all_hi >= first_key + 32;
        float2 part[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        auto tile = [&](auto whole_t) {
          constexpr bool WHOLE = decltype(whole_t)::value;
          float2 s[2][kRun / 2];
          tmem_ld16(ts + buf * 256, reinterpret_cast<uint32_t*>(s[0]));
          auto run = [&](float2 (&x)[kRun / 2], int j) {
            if (MODE & 1) cap_scores(x, c, cap2);
#pragma unroll
            for (int e = 0; e < kRun / 2; ++e) {
              const float2 l = *reinterpret_cast<const float2*>(&info.neg_lse[j + 2 * e]);
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
              }
              part[e & 1] = add2(part[e & 1], y);
            }
          };
#pragma unroll 1
          for (int j = 0; j < cols; j += 2 * kRun) {
            tmem_wait_ld();
            tmem_loaded<kRun>(reinterpret_cast<uint32_t*>(s[0]));
            const bool more = j + kRun < cols;
            if (more) tmem_ld16(ts + buf * 256 + j + kRun, reinterpret_cast<uint32_t*>(s[1]));
            run(s[0], j);
            if (more) {
              tmem_wait_ld();
              tmem_loaded<kRun>(reinterpret_cast<uint32_t*>(s[1]));
              if (j + 2 * kRun < cols) tmem_ld16(ts + buf * 256 + j + 2 * kRun, reinterpret_cast<uint32_t*>(s[0]));
              run(s[1], j + kRun);
            }
          }
        };
        if (!none) {
          if (whole) tile(std::true_type{});
          else tile(std::false_type{});
        }
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.s_empty[buf]);
        ++n_s;
        part[0] = add2(part[0], part[1]);
        sum = add2(sum, part[0]);
      }
      if (uniform(info.item.last) && mine + lane < info.item.room) {
        const long long at = info.item.h * w.slots + info.item.slot + key;
        const float x = sum.x + sum.y;
        if (w.partial) w.partial[info.item.part * w.slots * a.L.hkv + at] = x;
        else if (x != 0.f) w.weights[at] += x;
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
    tmem_free(tmem, 512);
  } else if (warp == 0) {
    // After a wait that ran out the CTA does not end under copies that nobody waited for.
    for (int i = max(0, sh.k_asked - P::kKRing); i < sh.k_asked; ++i)
      if (!warp_wait(&sh.k_full[i % P::kKRing], (i / P::kKRing) & 1, a.status)) break;
    for (int i = max(0, sh.q_asked - P::kQRing); i < sh.q_asked; ++i)
      if (!warp_wait(&sh.q_full[i % P::kQRing], (i / P::kQRing) & 1, a.status)) break;
  }
}

// What each chunk of w.tokens tokens sees, for masks that are given.
__global__ void __launch_bounds__(256) weigh_ranges_kernel(const WeighArgs w) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r = blockIdx.x;
  const Rows x = rows_of(w, r);
  const long long at = weigh_range_at(x.t.t0, r, w.tokens);
  for (int c = blockIdx.y * 8 + warp; c * w.tokens < x.n; c += gridDim.y * 8) {
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
  }
}

// weights += the parts' sums, in the order of the parts.
__global__ void __launch_bounds__(256) weigh_join_kernel(const WeighArgs w, int tiles) {
  const int tile = static_cast<int>(blockIdx.x % tiles);
  const int h = static_cast<int>(blockIdx.x / tiles) % w.a.L.hkv, r = static_cast<int>(blockIdx.x / tiles) / w.a.L.hkv;
  const Rows x = rows_of(w, r);
  const int key = tile * 256 + threadIdx.x;
  if (x.n == 0 || key >= x.t.len) return;
  const int parts = (x.tiles + w.per_part - 1) / w.per_part;
  const long long at = h * w.slots + static_cast<long long>(w.a.L.block_offsets[r]) * w.a.L.b + key;
  float sum = 0.f;
  for (int p = 0; p < parts; ++p) sum += w.partial[p * w.slots * w.a.L.hkv + at];
  w.weights[at] += sum;
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
  return r == CUDA_SUCCESS ? 0 : 1;
}

template <typename T, int D, int MODE>
int launch_mode(const WeighArgs& w, int sms, const CUtensorMap& km, const CUtensorMap& qm, cudaStream_t stream) {
  auto kern = weigh_tensor_kernel<T, D, MODE>;
  static_assert(sizeof(Shared<D>) <= 227 * 1024, "shared memory of a CTA");
  const int rc = static_cast<int>(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(Shared<D>)));
  if (rc) return rc;
  kern<<<sms, kThreads, sizeof(Shared<D>), stream>>>(w, km, qm);
  return static_cast<int>(cudaGetLastError());
}

template <typename T, int D>
int launch_d(const WeighArgs& w, int sms, const CUtensorMap& km, const CUtensorMap& qm, cudaStream_t stream) {
  switch ((w.a.softcap > 0.f ? 1 : 0) | (w.a.slopes ? 2 : 0)) {
    case 0: return launch_mode<T, D, 0>(w, sms, km, qm, stream);
    case 1: return launch_mode<T, D, 1>(w, sms, km, qm, stream);
    case 2: return launch_mode<T, D, 2>(w, sms, km, qm, stream);
    default: return launch_mode<T, D, 3>(w, sms, km, qm, stream);
  }
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
  int rc = encode_pool_map(&km, w.a, w.a.L.k, kv_dtype, w.a.L.page_size < 128 ? w.a.L.page_size : 128);
  if (rc) return rc;
  rc = encode_query_map(&qm, w, kv_dtype);
  if (rc) return rc;
  if (w.ranges) {
    weigh_ranges_kernel<<<dim3(w.a.R, 16), 256, 0, stream>>>(w);
    rc = static_cast<int>(cudaGetLastError());
    if (rc) return rc;
  }
  if (kv_dtype == kBF16)
    rc = w.a.d == 64 ? launch_d<__nv_bfloat16, 64>(w, sms, km, qm, stream) : launch_d<__nv_bfloat16, 128>(w, sms, km, qm, stream);
  else
    rc = w.a.d == 64 ? launch_d<__half, 64>(w, sms, km, qm, stream) : launch_d<__half, 128>(w, sms, km, qm, stream);
  if (rc || !w.partial) return rc;
  const int tiles = (w.longest + 255) / 256;
  const long long ctas = static_cast<long long>(tiles) * w.a.L.hkv * w.a.R;
  if (ctas > 0x7fffffff) return static_cast<int>(cudaErrorInvalidValue);
  weigh_join_kernel<<<static_cast<unsigned>(ctas), 256, 0, stream>>>(w, tiles);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace stk
