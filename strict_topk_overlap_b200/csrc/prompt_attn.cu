// Dense paged attention of many rows on the tensor cores (tcgen05): prompts,
// pieces of prompts, and all requests' tokens over a shared prefix.
//
// The rows of one KV head (new tokens x query heads of the group, packed) are
// cut into MMA tiles of 128, one or two to a CTA. Per 128 keys:
//   S = Q K^T          128 x 128, FP32 in tensor memory (TMEM)
//   P = 2^(c S - m)    two threads per row, 64 keys each: cap, bias, mask,
//                      running maximum and sum in FP32; P rounded to the type,
//                      over S in TMEM
//   O += P V           FP32 in TMEM, P the TMEM operand
// Warps 0-7 and 8-15 are the softmax of the two MMA tiles, warp 16 issues the
// MMAs (one tile's products run while the other tile's weights are formed),
// warp 17 feeds a ring of K and V tiles by TMA, one box per page and 64 dims,
// swizzled as the MMA reads them.
//
// Rounding: a weight is rounded to the type, by at most 2^-8 or 2^-11 of
// itself, as the output is. Scores, maxima, sums and O are FP32. The frame m
// of a row's weights may lie below its maximum: by up to 2^8, so that O is
// rescaled only when the maximum grew by more; bf16's range allows the growth
// of a whole tile on top, which saves a pass for the maximum (f16's does not).
//
// Tensor-bound in principle: 4 * 128 * 128 * D FLOP per 128 rows x 128 keys,
// 1,024 clocks at D = 128. In fact bound by the chain S -> P -> O of a tile:
// about 4,000 clocks per 256 rows x 128 keys, the tensor cores half idle. A
// tile's softmax is some 1,300 clocks of instructions when it has the SM to
// itself, and S cannot be formed again before P, which lies over it, is used
// (TMEM is full: two S and two O of 128 columns). Hence two MMA tiles, and
// each tile's keys in two halves with chains of their own, so that one's
// products run under another's exponentials.
//
// Measured (B200; calls in a row for seconds, where the power limit holds the
// clocks down, and in brackets short bursts): three causal prompts of 10.8 K
// tokens, 16 / 8 heads, D 128, capped: 300 (271) us, 746 TFLOP/s, plain (241);
// 509 tokens on 65 K keys, 32 / 8 heads, biased: 741 (690) us, 734 TFLOP/s,
// under half of cuBLAS's rate; 8 K tokens of packed documents, D 64, f16: 123
// us; prompts with prefix masks, 96 / 8 heads: 66 us. On the capped prompts, in
// bursts and in the order tried: MMAs issued under a branch on one lane 469 us,
// by a predicate 374 us; eight softmax warps with a row's 128 scores in
// registers 374 us, sixteen with 64 each 418 us (at 96 registers they spill,
// and 224 KB of shared memory leave next to no L1 for that), sixteen that keep
// the scores in TMEM 359 us; both halves of the keys in one chain 372 us, in
// two 343 us; the heads as the grid's slower dimension 334 us, innermost 267 us
// (the longest tiles of all heads start first). Even so 20 to 90 bytes a thread
// of what is used once per CTA spill.
//
// Tiles of keys that no row sees are not read; runs of 16 keys that a warp's
// rows all see skip the mask, those that none sees the exponentials. Places
// that no row of a CTA sees may hold anything, unwritten memory or unassigned
// table entries: pages of such keys alone read as zeros, and in pages that
// seen keys share K is masked and V zeroed in shared memory. A value that is
// not finite at a key some rows of a tile see and others do not turns the
// others' sums into NaN (0 * inf); such rows are recomputed one by one from
// their own keys.

#include "paged_tensor.cuh"
#include "tcgen05.cuh"

namespace stk {

int set_wait_limit_prompt(unsigned long long ns) { return set_wait_limit_this_unit(ns); }

namespace {

constexpr int kTileM = 128;   // rows of an MMA tile
constexpr int kTileN = 128;   // keys of a tile
constexpr float kLazy = 8.f;  // log2 of the growth of the maximum that is left to P

__device__ constexpr float kTanh3[3] = {0.99999961f, -0.33321959f, 0.1284243f};
__device__ constexpr float kTanh5[5] = {0.99999948f, -0.333285f, 0.13261181f, -0.05011862f, 0.012984885f};

struct Shared {
  uint64_t full[10], empty[10];
  uint64_t q_full[2], s_full[2][2], p_full[2][2], o_full[2];  // [MMA tile] or [MMA tile][half of the keys]
  uint64_t pair[8];            // the two warps that share 32 rows
  uint64_t drained;            // the products issued before a wait ran out
  volatile int abandoned;      // one of the MMA warp ran out
  volatile int asked;          // copies asked for when one of the load warp ran out, -1: all
  uint32_t tmem;
  int2 range[16];              // of a warp's rows: least and largest key
  volatile int failed[2];      // a wait of the MMA tile's softmax ran out
  union {
    float other[2][2][kTileM];             // [MMA tile][half of the keys][row]: maxima, at the end the sums
    unsigned short frame[2][4][kTileM];    // [MMA tile][key tile mod 4][row]: new frame less the tile's largest bias, upper half of its bits
  };
};
constexpr unsigned short kKeep = 0x7fc0;   // (a NaN) the frame stays

// Heads of 128 dims: two MMA tiles (256 rows) in a CTA that fills the SM, so
// that a K and V tile from L2 serves both. Heads of 64 dims need half the
// bytes and TMEM per MMA tile: one MMA tile in a CTA and two CTAs an SM, which
// start and end beside one another (packed documents 151 -> 146 us).
template <int D>
struct Plan {
  static constexpr int kMmaTiles = D == 128 ? 2 : 1;
  static constexpr int kRows = kMmaTiles * kTileM;
  static constexpr int kSoftmaxWarps = 8 * kMmaTiles;    // two groups of four per MMA tile, 64 keys each
  static constexpr int kThreads = (kSoftmaxWarps + 2) * 32;
  static constexpr int kCtas = 3 - kMmaTiles;            // per SM
  static constexpr int kTmem = 256 * kMmaTiles;          // columns: S, then O
  static constexpr int kTileBytes = kTileN * D * 2;      // one K or V tile, and one Q tile
  static constexpr int kQBytes = 32768;                  // a Q tile's place, at the end 4 KB of output for each warp
  static constexpr int kRing = D == 128 ? 5 : 4;         // K and V tiles in flight
  static constexpr int kBytes = kMmaTiles * kQBytes + kRing * kTileBytes + static_cast<int>(sizeof(Shared));
};

constexpr int kRun = 16;  // keys taken from TMEM at once

// What turns kRun raw scores S of a row into scores in log2 units: cap, bias
// and mask. Plain scores (MODE 0) stay raw, their factor joins the exponent.
struct Score {
  float c1;                  // scale * log2 e, or scale / cap
  float cap2;                // cap * log2 e
  float t0, t1, t2, t3, t4;  // cap2 c1^(2k + 1)
  float slope2;              // slope * log2 e
  RowKeys rk;
};

template <int MODE>
__device__ __forceinline__ void scores(float2 (&s)[kRun / 2], const Score& z, int k0, bool full) {
  // Capped scores cap2 tanh(c1 s) as odd polynomials in s (fitted for the
  // least relative error), no special functions: three terms where |c1 s| <=
  // 0.25 throughout a warp's run (4.3e-7), five up to 0.75 (6.3e-7), errors
  // of the order of FP32's own; the exponential form beyond.
  if (MODE & 1) {
    float far[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < kRun / 2; ++j) far[j & 1] = fmaxf(fmaxf(far[j & 1], fabsf(s[j].x)), fabsf(s[j].y));
    const float most = fmaxf(far[0], far[1]) * z.c1;
    if (__all_sync(kFull, most <= 0.25f)) {
      const float2 u0 = both(z.t0 * kTanh3[0]), u1 = both(z.t1 * kTanh3[1]), u2 = both(z.t2 * kTanh3[2]);
#pragma unroll
      for (int j = 0; j < kRun / 2; ++j) {
        const float2 y = mul2(s[j], s[j]);
        s[j] = mul2(s[j], fma2(y, fma2(y, u2, u1), u0));
      }
    } else if (__all_sync(kFull, most <= 0.75f)) {
      const float2 u0 = both(z.t0 * kTanh5[0]), u1 = both(z.t1 * kTanh5[1]), u2 = both(z.t2 * kTanh5[2]);
      const float2 u3 = both(z.t3 * kTanh5[3]), u4 = both(z.t4 * kTanh5[4]);
#pragma unroll
      for (int j = 0; j < kRun / 2; ++j) {
        const float2 y = mul2(s[j], s[j]);
        s[j] = mul2(s[j], fma2(y, fma2(y, fma2(y, fma2(y, u4, u3), u2), u1), u0));
      }
    } else {
#pragma unroll
      for (int j = 0; j < kRun / 2; ++j) s[j] = make_float2(z.cap2 * cap_tanh(s[j].x * z.c1), z.cap2 * cap_tanh(s[j].y * z.c1));
    }
  }
  if (MODE & 2) {
    // - slope |pos - k|: linear in k unless the run reaches past the row's place.
    const float c = (MODE & 1) ? 1.f : z.c1;
    const float at = static_cast<float>(k0 - z.rk.pos);
    if (__any_sync(kFull, k0 + kRun - 1 > z.rk.pos)) {
#pragma unroll
      for (int j = 0; j < kRun / 2; ++j) {
        s[j].x = fmaf(-z.slope2, fabsf(at + static_cast<float>(2 * j)), s[j].x * c);
        s[j].y = fmaf(-z.slope2, fabsf(at + static_cast<float>(2 * j + 1)), s[j].y * c);
      }
    } else {
      float2 away[2];  // every second pair's bias, four keys on at a time
#pragma unroll
      for (int x = 0; x < 2; ++x)
        away[x] = make_float2((at + static_cast<float>(2 * x)) * z.slope2, (at + static_cast<float>(2 * x + 1)) * z.slope2);
#pragma unroll
      for (int j = 0; j < kRun / 2; ++j) {
        s[j] = fma2(s[j], both(c), away[j & 1]);
        away[j & 1] = add2(away[j & 1], both(4.f * z.slope2));
      }
    }
  }
  if (!full) {
    const int lo = z.rk.lo - k0, hi = z.rk.hi - k0;
#pragma unroll
    for (int j = 0; j < kRun / 2; ++j) {
      s[j].x = 2 * j >= lo && 2 * j < hi ? s[j].x : neg_inf();
      s[j].y = 2 * j + 1 >= lo && 2 * j + 1 < hi ? s[j].y : neg_inf();
    }
  }
}

__device__ __forceinline__ float largest(const float2 (&s)[kRun / 2], float mx) {
  float top[2] = {mx, neg_inf()};
#pragma unroll
  for (int j = 0; j < kRun / 2; ++j) top[j & 1] = fmaxf(fmaxf(top[j & 1], s[j].x), s[j].y);
  return fmaxf(top[0], top[1]);
}

// Weights 2^(c s - m) of kRun keys, packed, and their sum.
template <typename T, int MODE, int FMA_PAIRS>
__device__ __forceinline__ void weights(const float2 (&s)[kRun / 2], float c, float nm, float2 (&sum)[2], uint32_t (&p)[kRun / 2]) {
#pragma unroll
  for (int e = 0; e < kRun / 2; ++e) {
    float2 x = MODE != 0 ? add2(s[e], both(nm)) : fma2(s[e], both(c), both(nm));
    x = (e & 7) < FMA_PAIRS ? ex2_fma(x) : make_float2(ex2(x.x), ex2(x.y));
    sum[e & 1] = add2(sum[e & 1], x);
    p[e] = pack2<T>(x.x, x.y);
  }
}

// MODE: 1 capped scores, 2 biased by distance, 3 both.
template <typename T, int D, int MODE>
__global__ void __launch_bounds__(Plan<D>::kThreads, Plan<D>::kCtas)
prompt_attn_kernel(const PagedAttnArgs a, const __grid_constant__ CUtensorMap kmap,
                   const __grid_constant__ CUtensorMap vmap) {
  using P = Plan<D>;
  constexpr int QT = P::kMmaTiles, kSoftmaxWarps = P::kSoftmaxWarps;
  constexpr bool kLag = std::is_same<T, __nv_bfloat16>::value;
  // Heads of 64 dims leave room in TMEM for an O of its own for each half of
  // the keys: the halves then share nothing until the end. Heads of 128 dims
  // share O, each half's warps keeping half of its dims in frame.
  constexpr bool kOwnO = D == 64;
  constexpr int kOCols = 64;  // of O, a warp's
  // Of 8 pairs of weights, those whose exponentials take the FMA units: two for
  // biased scores, whose frames move most (509 tokens on 65 K keys: 660 us, 672
  // with none); none for others (plain causal prompts of 10.8 K tokens 238 us,
  // 249 with two; 512 tokens on 16 K keys 149 against 159).
  constexpr int kFmaPairs = MODE == 2 ? 2 : 0;
  constexpr int kHalves = D / 64;
  constexpr int kHalfBytes = kTileN * 128;
  extern __shared__ __align__(1024) unsigned char base[];  // swizzle atoms: 1024-byte aligned
  unsigned char* ring = base + QT * P::kQBytes;
  Shared& sh = *reinterpret_cast<Shared*>(ring + P::kRing * P::kTileBytes);
  const int tid = threadIdx.x, lane = tid & 31, warp = uniform(tid >> 5);
  // Later row tiles see more keys under a causal mask: they start first, all
  // heads' together, so that the shortest end the grid.
  const int h = static_cast<int>(blockIdx.x) % a.L.hkv, rest = static_cast<int>(blockIdx.x) / a.L.hkv;
  const int slots = static_cast<int>(gridDim.x) / (a.L.hkv * a.nsplit);
  const int split = rest % a.nsplit;
  const RowTile t = row_tile<P::kRows>(a, slots - 1 - rest / a.nsplit, lane);
  if (t.rows == 0) return;

  const int qt = warp >> 3, half = (warp >> 2) & 1;        // softmax warps: MMA tile, half of its keys
  const int row = qt * kTileM + (tid & (kTileM - 1));      // and row of the CTA
  const bool have = row < t.rows;
  RowKeys rk{0, 0x7fffffff, 0};
  const int* table = nullptr;  // loads: the request's page table
  if (warp < kSoftmaxWarps) {
    const int my_tok = have ? (t.row0 + row) / a.G : 0;
    const int2 given = given_keys(a, t.t0 + my_tok);
    // Q tiles, swizzled: 16-byte chunk c of row x at chunk c ^ (x & 7). The copies run beside what follows.
    const T* q = static_cast<const T*>(a.q);
#pragma unroll
    for (int it = 0; it < D / 16; ++it) {
      const int x = it * 2 * kTileM + (tid & (2 * kTileM - 1));
      const int rr = x / (D / 8), c = x % (D / 8);
      const int cr = qt * kTileM + rr;
      unsigned char* dst = base + qt * P::kQBytes + (c >> 3) * kHalfBytes + rr * 128 + ((c ^ rr) & 7) * 16;
      if (cr < t.rows) {
        const int tok = (t.row0 + cr) / a.G, g = t.row0 + cr - tok * a.G;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)),
                     "l"(q + (t.t0 + tok) * a.q_ts + (h * a.G + g) * a.q_hs + c * 8)
                     : "memory");
      } else {
        *reinterpret_cast<uint4*>(dst) = make_uint4(0, 0, 0, 0);
      }
    }
    // The rows' key intervals.
    if (have) rk = row_keys(a, t, my_tok, given);
    const bool some = have && rk.hi > rk.lo;
    const int kmin = __reduce_min_sync(kFull, some ? rk.lo : 0x7fffffff);
    const int kmax = __reduce_max_sync(kFull, some ? rk.hi : 0);
    if (lane == 0) sh.range[warp] = make_int2(kmin, kmax);
  } else if (warp == kSoftmaxWarps) {
    tmem_alloc(&sh.tmem, P::kTmem);
  } else {
    table = a.L.page_table + static_cast<long long>(a.L.block_offsets[t.r]) * (a.L.b / a.L.page_size);
    if (lane == 0) {
      for (int i = 0; i < P::kRing; ++i) {
        mbar_init(&sh.full[i], 1);
        mbar_init(&sh.empty[i], 1);
      }
      for (int q = 0; q < QT; ++q) {
        mbar_init(&sh.q_full[q], 2 * kTileM);
        for (int x = 0; x < 2; ++x) {
          mbar_init(&sh.s_full[q][x], 1);
          mbar_init(&sh.p_full[q][x], kTileM);
        }
        mbar_init(&sh.o_full[q], 1);
        sh.failed[q] = 0;
      }
      for (int x = 0; x < 8; ++x) mbar_init(&sh.pair[x], 64);
      mbar_init(&sh.drained, 1);
      sh.abandoned = 0;
      sh.asked = -1;
      fence_barrier_init();
    }
    __syncwarp();
  }
  __syncthreads();
  // Each MMA tile's keys [kmin, kmax).
  int2 keys[2] = {make_int2(0x7fffffff, 0), make_int2(0x7fffffff, 0)};
  {
    int2 v = sh.range[lane & (kSoftmaxWarps - 1)];
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
      v.x = min(v.x, __shfl_xor_sync(kFull, v.x, o));
      v.y = max(v.y, __shfl_xor_sync(kFull, v.y, o));
    }
#pragma unroll
    for (int q = 0; q < QT; ++q) keys[q] = make_int2(__shfl_sync(kFull, v.x, 8 * q), __shfl_sync(kFull, v.y, 8 * q));
  }
  // Tiles [ta, tb) of this CTA's part, and those of each MMA tile.
  int ta, tb, qa[2] = {0, 0}, qb[2] = {0, 0};
  {
    const int kmin = min(keys[0].x, keys[1].x), kmax = max(keys[0].y, keys[1].y);
    const int first = kmax > 0 ? kmin / kTileN : 0, last = (kmax + kTileN - 1) / kTileN;
    const int per = (last - first + a.nsplit - 1) / a.nsplit;
    ta = min(last, first + split * per);
    tb = min(last, ta + per);
    int lo = tb, hi = ta;
#pragma unroll
    for (int q = 0; q < QT; ++q) {
      qa[q] = keys[q].y > 0 ? max(ta, keys[q].x / kTileN) : tb;
      qb[q] = min(tb, (keys[q].y + kTileN - 1) / kTileN);
      if (qb[q] <= qa[q]) qa[q] = qb[q] = ta;
      else {
        lo = min(lo, qa[q]);
        hi = max(hi, qb[q]);
      }
    }
    ta = uniform(lo);
    tb = uniform(max(lo, hi));
#pragma unroll
    for (int q = 0; q < QT; ++q) {
      qa[q] = uniform(qa[q]);
      qb[q] = uniform(qb[q]);
    }
  }
  // The keys that any row here sees lie in [.x, .y). (From shared memory once
  // more: the softmax warps have no registers to keep it in.)
  auto seen_keys = [&]() {
    const int2 v = sh.range[lane & (kSoftmaxWarps - 1)];
    return make_int2(__reduce_min_sync(kFull, v.x), __reduce_max_sync(kFull, v.y));
  };
  const uint32_t tmem = uniform(sh.tmem);
  const int rp = t.r;

  if (warp == kSoftmaxWarps + 1) {
    // ------------------------------------------------------------ K and V tiles
    const int bp = min(a.L.page_size, kTileN);  // rows of a box
    const int boxes = kTileN / bp;
    const int2 any = seen_keys();
    // Page of the box of keys from `key` on. Boxes of keys that no row here
    // sees read as zeros, whatever the table or the pool holds there; a bad
    // entry reads as zeros and is reported.
    auto page_at = [&](int key) {
      if (key >= any.y || key + bp <= any.x) return a.pages;
      const int page = table[key / a.L.page_size];
      if (page < 0 || page >= a.pages) {
        report(a.status, kStatusBadBlockId);
        return a.pages;
      }
      return page;
    };
    int page = lane < boxes && ta < tb ? page_at(ta * kTileN + lane * bp) : 0;
    bool ok = true;
    for (int i = ta; ok && i < tb; ++i) {
      const int next = lane < boxes && i + 1 < tb ? page_at((i + 1) * kTileN + lane * bp) : 0;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const int item = 2 * (i - ta) + kv, slot = item % P::kRing;
        if (item >= P::kRing) ok = ok && warp_wait(&sh.empty[slot], (item / P::kRing - 1) & 1, a.status);
        if (!ok) {
          sh.asked = item;
          break;
        }
        if (lane == 0) mbar_arrive_expect_tx(&sh.full[slot], P::kTileBytes);
        __syncwarp();
        if (lane < boxes) {
          unsigned char* dst = ring + slot * P::kTileBytes + lane * bp * 128;
          const int y = (i * kTileN + lane * bp) % a.L.page_size;
#pragma unroll
          for (int half = 0; half < kHalves; ++half)
            tma_load(kv == 0 ? &kmap : &vmap, dst + half * kHalfBytes, &sh.full[slot], half * 64, y, h, page);
        }
      }
      page = next;
    }
  } else if (warp == kSoftmaxWarps) {
    // ------------------------------------------------------------ MMAs
    constexpr uint32_t qk = mma_desc<T>(kTileM, kTileN / 2, false), pv = mma_desc<T>(kTileM, D, true);
    const uint64_t q_desc = smem_desc(smem_u32(base), 16), k_desc = smem_desc(smem_u32(ring), 16);
    const uint64_t v_desc = smem_desc(smem_u32(ring), kHalfBytes);
    constexpr uint64_t kTile16 = P::kTileBytes >> 4;  // descriptor addresses count 16 bytes
    const int2 any = seen_keys();
    int done[2] = {0, 0};  // tiles, per MMA tile
    // Ring slots and phases of the next K and V tiles (items 0, 2, 4, .. and 1, 3, 5, ..).
    int slot = 0, phase = 0;
    auto advance = [&]() {
      if (++slot == P::kRing) {
        slot = 0;
        phase ^= 1;
      }
    };
    auto issue_qk = [&](int q, int x, int kslot) {  // S = Q K^T, half x of the keys
      const uint64_t kd = k_desc + kslot * kTile16 + x * (kHalfBytes / 2 >> 4), qd = q_desc + q * (P::kQBytes >> 4);
#pragma unroll
      for (int s = 0; s < D / 16; ++s) {
        const uint64_t o = ((s >> 2) * kHalfBytes + (s & 3) * 32) >> 4;
        mma_ss(tmem + q * kTileN + x * (kTileN / 2), qd + o, kd + o, qk, s > 0);
      }
      mma_commit(&sh.s_full[q][x]);
    };
    bool ok = true;
    if (ta < tb) {
      ok = warp_wait(&sh.full[0], 0, a.status);
#pragma unroll
      for (int q = 0; q < QT; ++q) {
        if (qa[q] < qb[q]) ok = ok && warp_wait(&sh.q_full[q], 0, a.status);
        fence_after();
        if (ok && qa[q] == ta && qa[q] < qb[q]) {
          issue_qk(q, 0, 0);
          issue_qk(q, 1, 0);
        }
      }
      mma_commit(&sh.empty[0]);
      advance();
    }
    for (int i = ta; ok && i < tb; ++i) {
      const int vslot = slot;
      ok = warp_wait(&sh.full[vslot], phase, a.status);
      if (!ok) break;
      // Keys that no row here sees, in pages that others of theirs share:
      // their values must not meet the zero weights.
      const int from = any.x - i * kTileN, to = any.y - i * kTileN;
      if (from > 0 || to < kTileN) {
        // Below `from` and from `to` on, each to the end of its box.
        unsigned char* vt = ring + vslot * P::kTileBytes;
        const int bp = min(a.L.page_size, kTileN);
        const int below = max(from, 0) % bp, above = to < kTileN ? (bp - to % bp) % bp : 0;
#pragma unroll 1
        for (int x = lane; x < (below + above) * 8 * kHalves; x += 32) {
          const int half = x % kHalves, c = x / kHalves % 8, y = x / (8 * kHalves);
          const int at = y < below ? from - below + y : to + y - below;
          *reinterpret_cast<uint4*>(vt + half * kHalfBytes + at * 128 + c * 16) = make_uint4(0, 0, 0, 0);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
      }
      advance();
      const int kslot = slot;
      const bool more = i + 1 < tb;
      if (more) ok = warp_wait(&sh.full[kslot], phase, a.status);
#pragma unroll
      for (int q = 0; q < QT; ++q) {
        const bool now = i >= qa[q] && i < qb[q], then = i + 1 >= qa[q] && i + 1 < qb[q];
        const uint64_t vd = v_desc + vslot * kTile16;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (ok && now) {  // O += P V
            ok = warp_wait(&sh.p_full[q][x], done[q] & 1, a.status);
            fence_after();
#pragma unroll
            for (int s = 0; s < kTileN / 32; ++s)
              mma_ts(tmem + QT * kTileN + (kOwnO ? q * 2 + x : q * 2) * kOCols, tmem + q * kTileN + x * (kTileN / 2) + s * 8,
                     vd + (x * (kTileN / 32) + s) * (2048 >> 4), pv, done[q] > 0 || (!kOwnO && x > 0) || s > 0);
          }
          if (ok && then) issue_qk(q, x, kslot);
        }
        if (now) {
          if (i + 1 == qb[q]) mma_commit(&sh.o_full[q]);
          ++done[q];
        }
      }
      mma_commit(&sh.empty[vslot]);
      if (more) {
        mma_commit(&sh.empty[kslot]);
        advance();
      }
    }
    if (!ok) {  // a wait ran out and was reported: tensor memory is freed after the products under way
      sh.abandoned = 1;
      mma_commit(&sh.drained);
      warp_wait(&sh.drained, 0, a.status);
    }
  } else if (warp < kSoftmaxWarps) {
    // ------------------------------------------------------------ softmax
    constexpr int kKeys = kTileN / 2;  // of a thread
    const int r = tid & (kTileM - 1);  // row of the MMA tile
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // TMEM lane 32 (warp % 4)
    const uint32_t ts = tmem + lanes + qt * kTileN + half * kKeys;
    const uint32_t to = tmem + lanes + QT * kTileN + (qt * 2 + half) * kOCols;
    asm volatile("cp.async.wait_all;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    mbar_arrive(&sh.q_full[qt]);
    // What the warp's 32 rows see of a run of keys: nothing (no weights to form), all of it (no mask), or some.
    enum { kNone, kSome, kAll };
    const int lo_min = __reduce_min_sync(kFull, have ? rk.lo : 0x7fffffff), lo_max = __reduce_max_sync(kFull, rk.lo);
    const int hi_max = __reduce_max_sync(kFull, have ? rk.hi : 0), hi_min = __reduce_min_sync(kFull, rk.hi);
    auto seen = [&](int k) {
      return k + kRun <= lo_min || k >= hi_max ? kNone : k >= lo_max && k + kRun <= hi_min ? kAll : kSome;
    };
    const int tok = have ? (t.row0 + row) / a.G : 0;
    const int head = h * a.G + (have ? t.row0 + row - tok * a.G : 0);
    const float slope = (MODE & 2) && a.slopes ? a.slopes[head] : 0.f;
    Score z;
    z.c1 = (MODE & 1) ? a.scale / a.softcap : a.scale * kLog2e;
    z.cap2 = a.softcap * kLog2e;
    z.slope2 = slope * kLog2e;
    z.rk = rk;
    const float cc = z.c1 * z.c1;
    z.t0 = z.cap2 * z.c1;
    z.t1 = z.t0 * cc;
    z.t2 = z.t1 * cc;
    z.t3 = z.t2 * cc;
    z.t4 = z.t3 * cc;
    const float c = MODE != 0 ? 1.f : z.c1;
    float m = neg_inf(), l = 0.f;  // in log2 units; m is the frame of P, O and l, near the row's maximum
    bool ok = true, exact = true;
    int meetings = 0;
    float level = neg_inf();  // the scores' maximum so far, or a little more, less the bias
    const int begin = qt ? qa[1] : qa[0], end = qt ? qb[1] : qb[0];
    // O of the warp's rows (this half of its dims) and l by 2^(m - frame).
    auto reframe = [&](bool grow, float frame) {
      const float f = grow ? ex2(m - frame) : 1.f;
      l *= f;
#pragma unroll 1
      for (int j = 0; j < kOCols; j += 32) {
        uint32_t o[32];
        tmem_ld32(to + j, o);
        tmem_wait_ld();
        tmem_loaded(o);
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
        tmem_st32(to + j, o);
      }
      tmem_wait_st();
      fence_before();
      if (grow) m = frame;
    };
    // The two warps of the same rows: neither's next P is announced before both have been here.
    auto meet = [&]() {
      uint64_t* bar = &sh.pair[qt * 4 + (warp & 3)];
      fence_before();
      mbar_arrive(bar);
      ok = warp_wait(bar, meetings & 1, a.status) && ok;
      fence_after();  // the other's products and its accesses to O come before ours from here on
      ++meetings;
    };
    // P of the thread's keys from k0 on, over S, and their sum. WHOLE: every
    // row of the warp sees all of them, one straight run of code; else run by
    // run. RAW: S are still raw scores. The next run is on its way from TMEM
    // while one is computed.
    auto form_weights = [&](auto whole_t, auto raw_t, int k0, float nm, float2 (&sum)[2]) {
      constexpr bool WHOLE = decltype(whole_t)::value, RAW = decltype(raw_t)::value;
      float2 s[2][kRun / 2];
      tmem_ld16(ts, reinterpret_cast<uint32_t*>(s[0]));
#pragma unroll
      for (int j = 0; j < kKeys / kRun; ++j) {
        uint32_t p[kRun / 2];
        tmem_wait_ld();
        tmem_loaded<kRun>(reinterpret_cast<uint32_t*>(s[j & 1]));
        if (j + 1 < kKeys / kRun) tmem_ld16(ts + (j + 1) * kRun, reinterpret_cast<uint32_t*>(s[(j + 1) & 1]));
        const int view = WHOLE ? static_cast<int>(kAll) : seen(k0 + j * kRun);
        if (!WHOLE && view == kNone) {
#pragma unroll
          for (int e = 0; e < kRun / 2; ++e) p[e] = 0u;
        } else {
          if (RAW) scores<MODE>(s[j & 1], z, k0 + j * kRun, view == kAll);
          weights<T, MODE, kFmaPairs>(s[j & 1], c, nm, sum, p);
        }
        tmem_st8(ts + j * kRun / 2, p);  // over scores that have been read
      }
    };
    auto grows = [&](float x) { return x > m + kLazy || (m == neg_inf() && x > m); };
    // The bias of key `last`, or of the row's last key before it: the largest of a run that ends there.
    auto bias_at = [&](int last) {
      return (MODE & 2) ? -z.slope2 * static_cast<float>(max(0, rk.pos - min(last, rk.hi - 1))) : 0.f;
    };
    auto half_bias = [&](int i) { return bias_at(i * kTileN + half * kKeys + kKeys - 1); };  // of this thread's keys
    auto tile_bias = [&](int i) { return bias_at(i * kTileN + kTileN - 1); };
    for (int i = begin; i < end; ++i) {
      const int n = i - begin;
      // A wait that runs out is told to the whole group at its next meeting: nobody is left waiting there.
      ok = warp_wait(&sh.s_full[qt][half], n & 1, a.status) && ok;
      if (!ok) sh.failed[qt] = 1;
      if (kOwnO && !ok) break;
      fence_after();
      const int k0 = i * kTileN + half * kKeys;
      float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      const bool whole = k0 >= lo_max && k0 + kKeys <= hi_min, was_exact = exact;
      float est = 0.f;
      if (exact) {
        // The maximum first, over both halves of the row's keys. Transformed and masked scores go back to TMEM.
        float mx = neg_inf();
        bool wrote = false;
        float2 s[kRun / 2];
#pragma unroll 1
        for (int j0 = 0; j0 < kKeys; j0 += kRun) {
          const int view = seen(k0 + j0);
          if (view == kNone) continue;
          tmem_ld16(ts + j0, reinterpret_cast<uint32_t*>(s));
          tmem_wait_ld();
          tmem_loaded<kRun>(reinterpret_cast<uint32_t*>(s));
          scores<MODE>(s, z, k0 + j0, view == kAll);
          if (MODE != 0 || view != kAll) {
            tmem_st16(ts + j0, reinterpret_cast<const uint32_t*>(s));
            wrote = true;
          }
          mx = largest(s, mx);
        }
        if (wrote) tmem_wait_st();
        mx *= c;
        // (Read before this thread's P is announced, and written again after the next S, which waits for that.)
        if (!kOwnO) sh.other[qt][half][r] = mx;
        if (kOwnO) {
          const bool grow = grows(mx);
          if (__any_sync(kFull, grow && m != neg_inf())) reframe(grow, mx);
          else if (grow) m = mx;
        } else if (group_any(QT == 1 ? 1 : 1 + qt, 2 * kTileM, grows(mx) || !ok)) {
          if (sh.failed[qt]) {
            ok = false;
            break;
          }
          mx = fmaxf(mx, sh.other[qt][half ^ 1][r]);
          // Both halves' products are complete, their S come after them.
          const bool grow = grows(mx);
          if (__any_sync(kFull, grow && m != neg_inf())) reframe(grow, mx);
          else if (grow) m = mx;
          group_any(QT == 1 ? 1 : 1 + qt, 2 * kTileM, false);
        }
        const float nm = m == neg_inf() ? 0.f : -m;
        if (whole) form_weights(std::true_type{}, std::false_type{}, k0, nm, sum);
        else form_weights(std::false_type{}, std::false_type{}, k0, nm, sum);
        // Once every row that sees a key in this part has met one, the frames may lag (not f16's: P would leave its range).
        const bool waiting = m == neg_inf() && rk.hi > (i + 1) * kTileN && rk.lo < end * kTileN;
        if (kLag) exact = kOwnO ? __any_sync(kFull, waiting) : group_any(QT == 1 ? 1 : 1 + qt, 2 * kTileM, waiting);
      } else {
        // One pass, without a maximum, in a frame that the first half of the
        // keys sets at the end of the tile before: P may exceed 1, which
        // bf16's range and relative precision do not mind. The two halves of a
        // row are two independent chains of S, P and O that meet only where
        // the frame moves. A row whose scores run ahead of its frame by more
        // than 2^100 at the end is recomputed like those below.
        if (kOwnO) {
          const float frame = level + half_bias(i);
          const bool grow = grows(frame);
          if (__any_sync(kFull, grow)) reframe(grow, frame);
        } else {
          const unsigned short code = sh.frame[qt][n & 3][r];
          const bool grow = code != kKeep;
          const float frame = __uint_as_float(static_cast<uint32_t>(code) << 16) + tile_bias(i);
          if (__any_sync(kFull, grow)) {
            meet();  // both halves' products of the last tile are complete
            reframe(grow, frame);
            meet();
          }
        }
        const float nm = m == neg_inf() ? 0.f : -m;
        if (whole) form_weights(std::true_type{}, std::true_type{}, k0, nm, sum);
        else form_weights(std::false_type{}, std::true_type{}, k0, nm, sum);
        est = log2f((sum[0].x + sum[1].x) + (sum[0].y + sum[1].y)) - nm;  // the maximum, or a little more
      }
      // The next tile's frame: the level of the scores without their bias, and
      // the largest bias that the row meets there, so that a bias which grows
      // from tile to tile is followed at once. Keys too far below the frame to
      // weigh anything say nothing of the level.
      if (m == neg_inf()) level = neg_inf();
      else if (was_exact) level = m - (kOwnO ? half_bias(i) : tile_bias(i));
      else if (est - m > -100.f) level = est - half_bias(i);
      if (kLag && !kOwnO && half == 0 && !exact) {
        // Rounded down: a frame above the maximum would lose weights, one below it costs range only.
        const uint32_t code = (__float_as_uint(level) + (level < 0.f ? 0xffffu : 0u)) >> 16;
        const bool grow = m != neg_inf() && grows(__uint_as_float(code << 16) + tile_bias(i + 1));
        sh.frame[qt][(n + 1) & 3][r] = grow ? static_cast<unsigned short>(code) : kKeep;
      }
      tmem_wait_st();
      fence_before();
      mbar_arrive(&sh.p_full[qt][half]);
      sum[0] = add2(sum[0], sum[1]);
      l += sum[0].x + sum[0].y;
      if (!ok) break;
    }
    // ------------------------------------------------------------ output
    pdl_release();  // what follows in the call may be launched: a join waits for the states, a second phase for nothing
    const bool any = begin < end;
    if (any) ok = warp_wait(&sh.o_full[qt], 0, a.status) && ok;
    fence_after();
    // The row's two threads meet once. A shared O: its sum over both halves of
    // the keys. An O of its own for each half: the second half's thread hands
    // its state to the first's, through the ring, which is free now.
    float* handed = reinterpret_cast<float*>(ring + r * 256);  // 16-byte chunk c of row r at chunk c ^ (r & 7)
    if (kOwnO && half && ok) {
#pragma unroll 1
      for (int j = 0; j < kOCols; j += 32) {
        uint32_t o[32];
        if (any) {
          tmem_ld32(to + j, o);
          tmem_wait_ld();
          tmem_loaded(o);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e)
          *reinterpret_cast<uint4*>(handed + (((j / 4 + e) ^ (r & 7)) * 4)) =
              any ? make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]) : make_uint4(0, 0, 0, 0);
      }
      reinterpret_cast<float*>(ring + kTileM * 256)[r] = m;
    }
    sh.other[qt][half][r] = l;
    ok = !group_any(QT == 1 ? 1 : 1 + qt, 2 * kTileM, !ok);
    const float l2 = sh.other[qt][half ^ 1][r];
    float mine = 1.f, others = 0.f;
    const bool nan = l != l || l2 != l2;
    if (kOwnO) {
      const float m2 = half ? neg_inf() : reinterpret_cast<const float*>(ring + kTileM * 256)[r];
      const float frame = fmaxf(m, m2);
      mine = m == neg_inf() ? 0.f : ex2(m - frame);
      others = m2 == neg_inf() ? 0.f : ex2(m2 - frame);
      l = (mine == 0.f ? 0.f : l * mine) + (others == 0.f ? 0.f : l2 * others);
      m = frame;
    } else {
      l += l2;
    }
    const bool empty = m == neg_inf();
    const long long orow = static_cast<long long>(t.t0 + tok) * a.hq + head;
    const long long prow = static_cast<long long>(split) * a.T * a.hq + orow;
    const float inv = empty || a.part_ml ? 1.f : 1.f / l;
    // The frame was left behind, or ahead, by so much that sums of large values
    // may have left FP32's range (2^100; a frame that follows stays far inside);
    // or scores are NaN, perhaps all that the row sees here (which leaves no
    // maximum). The row's state is then taken anew in a frame of its own.
    const bool sees = have && max(rk.lo, begin * kTileN) < min(rk.hi, end * kTileN);
    const bool over = sees && (empty || nan || !(l <= 1.3e30f && l >= 7.9e-31f));
    bool redo_row = over;
    if (ok && !(kOwnO && half)) {
      // 128 bytes a row at a time through this warp's share of the Q tile's
      // place, which is free now, so that a store instruction covers whole rows.
      unsigned char* stage = base + qt * P::kQBytes + (warp & 7) * 4096;
      auto put = [&](int c, uint4 w) {  // 16-byte chunk c of the lane's row
        *reinterpret_cast<uint4*>(stage + lane * 128 + ((c ^ lane) & 7) * 16) = w;
      };
      // The staged rows to byte `at` of their rows of `stride` bytes.
      auto flush = [&](unsigned char* to, long long my_row, long long stride, int at) {
        __syncwarp();
        const int c = lane & 7;
        for (int r0 = 0; r0 < 32; r0 += 4) {
          const int rr = r0 + lane / 8;
          const long long dst = __shfl_sync(kFull, my_row, rr);
          const uint4 w = *reinterpret_cast<const uint4*>(stage + rr * 128 + ((c ^ rr) & 7) * 16);
          if (__shfl_sync(kFull, static_cast<int>(have), rr))
            *reinterpret_cast<uint4*>(to + dst * stride + at + c * 16) = w;
        }
        __syncwarp();
      };
      const int first_dim = kOwnO ? 0 : half * kOCols;
#pragma unroll 1
      for (int j = 0; j < kOCols; j += 32) {
        uint32_t o[32];
        if (any) {
          tmem_ld32(to + j, o);
          tmem_wait_ld();
          tmem_loaded(o);
        }
        if (kOwnO) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float4 y = *reinterpret_cast<const float4*>(handed + (((j / 4 + e) ^ (r & 7)) * 4));
            auto sum = [&](uint32_t x, float z) {
              return __float_as_uint((mine == 0.f ? 0.f : __uint_as_float(x) * mine) + (others == 0.f ? 0.f : z * others));
            };
            o[4 * e] = sum(o[4 * e], y.x);
            o[4 * e + 1] = sum(o[4 * e + 1], y.y);
            o[4 * e + 2] = sum(o[4 * e + 2], y.z);
            o[4 * e + 3] = sum(o[4 * e + 3], y.w);
          }
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float f = !any || empty ? 0.f : __uint_as_float(o[e]) * inv;
          redo_row = redo_row || (have && !(fabsf(f) <= 3.0e38f));
          o[e] = __float_as_uint(f);
        }
        if (a.part_ml) {
#pragma unroll
          for (int e = 0; e < 8; ++e) put(e, make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]));
          flush(reinterpret_cast<unsigned char*>(a.part_o), prow, D * 4, (first_dim + j) * 4);
        } else {
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) w[e] = pack2<T>(__uint_as_float(o[2 * e]), __uint_as_float(o[2 * e + 1]));
#pragma unroll
          for (int e = 0; e < 4; ++e)
            put((j & 32) / 8 + e, make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]));
          if (j) flush(static_cast<unsigned char*>(a.out), orow, D * 2, first_dim * 2);
        }
      }
      if (have && half == 0) {
        if (a.part_ml) a.part_ml[prow] = make_float2(empty ? neg_inf() : m * kLn2, l);
        else if (a.lse) a.lse[orow] = empty ? neg_inf() : (m + log2f(l)) * kLn2;
      }
      // Rows whose sums are not finite, be it for values of keys that they may
      // not see: this half of their dims once more, in the frame (m, l) that
      // stands, or in their own where l itself is lost.
      unsigned redo = __ballot_sync(kFull, redo_row);
      while (redo) {
        const int src = __ffs(redo) - 1;
        redo &= redo - 1;
        __syncwarp();
        const int xtok = __shfl_sync(kFull, tok, src);
        const int xhead = __shfl_sync(kFull, head, src), xpos = __shfl_sync(kFull, rk.pos, src);
        const int xlo = max(__shfl_sync(kFull, rk.lo, src), begin * kTileN);
        const int xhi = min(__shfl_sync(kFull, rk.hi, src), end * kTileN);
        const float xslope = __shfl_sync(kFull, slope, src);
        const float frame = __shfl_sync(kFull, m, src) * kLn2;
        const bool lost = __shfl_sync(kFull, static_cast<int>(over), src) != 0;
        float xm, xl, xo[D / 32];
        single_row<T, D>(a, rp, h, static_cast<const T*>(a.q) + (t.t0 + xtok) * a.q_ts + xhead * a.q_hs, xlo, xhi,
                         xpos, xslope, lane, xm, xl, xo);
        const long long xr = static_cast<long long>(t.t0 + xtok) * a.hq + xhead;
        const long long xp = static_cast<long long>(split) * a.T * a.hq + xr;
        const float factor = !a.part_ml ? (xl == 0.f ? 0.f : 1.f / xl) : lost ? 1.f : expf(xm - frame);
        if (lost && half == 0 && lane == 0) {
          if (a.part_ml) a.part_ml[xp] = make_float2(xm, xl);
          else if (a.lse) a.lse[xr] = xm + logf(xl);
        }
        if (kOwnO || (lane >> 4) == half) {
#pragma unroll
          for (int j = 0; j < D / 32; ++j) {
            const int dd = lane * (D / 32) + j;
            if (a.part_ml) a.part_o[xp * D + dd] = xo[j] * factor;
            else static_cast<unsigned short*>(a.out)[xr * D + dd] = static_cast<unsigned short>(pack2<T>(xo[j] * factor, 0.f));
          }
        }
      }
    }
    fence_before();
  }
  __syncthreads();
  if (warp == kSoftmaxWarps) {
    fence_after();
    tmem_free(sh.tmem, P::kTmem);
  }
  if (warp == kSoftmaxWarps + 1 && sh.abandoned) {  // the CTA does not end under copies that nobody waited for
    const int asked = sh.asked >= 0 ? sh.asked : 2 * (tb - ta);
    for (int item = max(0, asked - P::kRing); item < asked; ++item)
      if (!warp_wait(&sh.full[item % P::kRing], (item / P::kRing) & 1, a.status)) break;
  }
}

template <typename T, int D, int MODE>
int launch_mode(const PagedAttnArgs& a, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t stream) {
  auto kern = prompt_attn_kernel<T, D, MODE>;
  const int rc = static_cast<int>(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Plan<D>::kBytes));
  if (rc) return rc;
  const int slots = row_tile_slots(a.R, a.T, a.G, a.token_offsets != nullptr, a.shared != 0, Plan<D>::kRows);
  const long long ctas = static_cast<long long>(slots) * a.nsplit * a.L.hkv;
  if (ctas > 0x7fffffff) return static_cast<int>(cudaErrorInvalidValue);
  kern<<<static_cast<unsigned>(ctas), Plan<D>::kThreads, Plan<D>::kBytes, stream>>>(a, km, vm);
  return static_cast<int>(cudaGetLastError());
}

template <typename T, int D>
int launch_d(const PagedAttnArgs& a, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t stream) {
  switch ((a.softcap > 0.f ? 1 : 0) | (a.slopes ? 2 : 0)) {
    case 0: return launch_mode<T, D, 0>(a, km, vm, stream);
    case 1: return launch_mode<T, D, 1>(a, km, vm, stream);
    case 2: return launch_mode<T, D, 2>(a, km, vm, stream);
    default: return launch_mode<T, D, 3>(a, km, vm, stream);
  }
}

}  // namespace

// 16-bit types, heads of 64 or 128 dims, pages that tile 128 keys (or are
// tiled by them), 16-byte rows.
bool prompt_attn_takes(int kv_dtype, int d, int page_size, const void* k, const void* v, const void* q, long long q_ts,
                       long long q_hs, const void* out) {
  const bool pages = page_size >= 8 && (page_size <= kTileN ? kTileN % page_size == 0 : page_size % kTileN == 0);
  const uintptr_t any = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(q) |
                        reinterpret_cast<uintptr_t>(out) | static_cast<uintptr_t>(q_ts * 2) | static_cast<uintptr_t>(q_hs * 2);
  return kv_dtype != kF32 && (d == 64 || d == 128) && pages && any % 16 == 0;
}

int launch_prompt_attn(const PagedAttnArgs& a, int kv_dtype, cudaStream_t stream) {
  CUtensorMap km, vm;
  const int rows = a.L.page_size < kTileN ? a.L.page_size : kTileN;
  int rc = encode_pool_map(&km, a, a.L.k, kv_dtype, rows);
  if (rc == 0) rc = encode_pool_map(&vm, a, a.L.v, kv_dtype, rows);
  if (rc) return rc;
  if (kv_dtype == kBF16)
    return a.d == 64 ? launch_d<__nv_bfloat16, 64>(a, km, vm, stream) : launch_d<__nv_bfloat16, 128>(a, km, vm, stream);
  return a.d == 64 ? launch_d<__half, 64>(a, km, vm, stream) : launch_d<__half, 128>(a, km, vm, stream);
}

}  // namespace stk
