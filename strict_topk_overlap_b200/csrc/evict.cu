// Eviction from a paged cache: of each request's KV head the tokens of the
// largest weights stay (ties to the lower place; the first and last ones are
// protected), in their order, at the front of the request's own pages.
//
// Selection: a row (request, KV head) lies in the shared memory of a cluster
// of up to eight CTAs, read once. The threshold's bin is found in a histogram over
// the distance of the weights' order keys from the largest one, 32 bins to an
// octave, and its tokens are sorted by one CTA, one to a thread (zeros have a bin
// of their own and need no sorting). What is left crowded (equal weights) is
// found digit by digit of the order keys. Then every warp counts and writes its
// stretch in order: IDs, weights and, for the move, how many kept tokens lie
// before each chunk.
//
// Move: kept token i goes to place i <= its own. Moving in place saves half the
// bytes of a way through a copy, but a place may be overwritten only after it
// has been read. A warp copies a chunk into shared memory, announces that, waits
// for the (at most two) earlier chunks that read the places it writes, and writes.
// The warps of a co-resident grid take chunks in ascending order, so each waits
// for earlier ones only and some warp can always go on. As many warps as shared
// memory holds chunks for: each is a chain of latencies (places, rows, the
// announcement, the wait). A block's key bounds are taken by the warp that moves
// its keys.
//
// Measured (B200, D 128, calls in a row): 16 prompts of 1.5-32 K tokens cut to
// 2 K each, 8 heads, bf16 (268 MB moved, 120 MB of bounds reset): 114 us, 52 of
// them the selection, whose CTAs hold 32 K weights each; 6 requests of 20-60 K
// tokens cut to 16 K, f16 (800 MB moved): 212 us, 4 TB/s; 6 requests of 8-9 K
// to 4 K, FP32: 131. Read and written rows are single ones of 256 bytes wherever
// the kept tokens lie. The first two calls with 12 warps an SM of two chunks each
// took 126 and 240 us, 14: 118 and 224, chunks of 16 rows 146 and 268, chunks in
// registers and one item for every block of the cache, kept or not, 199 and 309;
// the selection by three passes of digits instead of one histogram 48 instead of
// 30 us (without the bounds), by twice the CTAs, two to an SM, the same; emptied
// blocks' bounds reset by the move's warps 113 and 214, the FP32 call 135. A copy to
// other pages and back would move twice the bytes.

#include <cooperative_groups.h>

#include <type_traits>

#include "cta_select.cuh"
#include "evict.cuh"

namespace stk {

int set_wait_limit_evict(unsigned long long ns) { return set_wait_limit_this_unit(ns); }

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 1024, kBins = 1024;  // one bin to a thread
constexpr int kBinShift = 18;                 // 32 bins to an octave
constexpr float kNothing = 1e30f;             // lo, and minus hi, of a block without tokens

// Weights in ascending order, NaN above all, zeros of either sign alike.
__device__ __forceinline__ uint32_t weight_key(float x) { return x == x ? order_key(x) : 0xffffffffu; }

// Tokens of request r, at most as many as its blocks hold.
__device__ __forceinline__ int held_tokens(const EvictArgs& a, int r) {
  const int n = a.lengths[r], room = min(request_blocks(a.L, r) * a.L.b, a.longest);
  if (n < 0 || n > room) report(a.status, kStatusBadLength);
  return max(0, min(n, room));
}

struct SelectShared {
  int hist[2][kBins];   // of two passes by turns: a sibling may still read the last one's
  u64 list[kThreads];   // tokens of a bin: weight key, and the place's complement
  uint2 kinds[kEvictSlice / 32];  // of each 32 tokens: which stay, which are at the threshold
  int warp_sums[32];
  uint32_t warp_top[32];
  uint32_t top;         // of the CTA: the largest key
  int2 count;           // tokens above the threshold (or protected), tokens at it
  int bin, above, crowd, listed;
  uint32_t limit;
  int take;
};

__global__ void __launch_bounds__(kThreads, 1) evict_select_kernel(const EvictArgs a) {
  extern __shared__ __align__(16) float row[];
  __shared__ SelectShared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = static_cast<int>(cluster.num_blocks()), part = static_cast<int>(cluster.block_rank());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int id = static_cast<int>(blockIdx.x) / parts, r = id / a.L.hkv, h = id - r * a.L.hkv;
  const int len = held_tokens(a, r), room = request_blocks(a.L, r) * a.L.b, now = min(len, a.keep);
  const long long base = h * a.slots + static_cast<long long>(a.L.block_offsets[r]) * a.L.b;
  const float* weights = a.weights + base;
  float* out = a.weights_out + base;
  int* kept = a.kept + static_cast<long long>(id) * a.keep;
  const int all = parts * kThreads, at = part * kThreads + tid;
  if (h == 0 && at == 0) a.lengths_out[r] = now;
  if (len <= a.keep) {  // everything stays
    for (int i = at; i < a.keep; i += all) kept[i] = i < len ? i : -1;
    if (out != weights)
      for (int i = at; i < len; i += all) out[i] = weights[i];
    for (int i = len + at; i < room; i += all) out[i] = 0.f;
    return;
  }
  int* rank = a.rank + static_cast<long long>(id) * (a.chunks + 1);
  int* read = a.read + static_cast<long long>(id) * 2 * a.segments * a.chunks;
  for (int i = at; i < 2 * a.segments * a.chunks; i += all) read[i] = 0;

  // ---- the CTA's slice [begin, end) of the row, whole groups of 32
  const int slice = ((len + parts - 1) / parts + 31) / 32 * 32;
  const int begin = min(len, part * slice), end = min(len, begin + slice), n = end - begin;
  const int lo = a.first, hi = len - a.last;  // the others of the row are protected
  uint32_t top = 0;
  auto look = [&](int i, float x) {
    if (begin + i >= lo && begin + i < hi) top = max(top, weight_key(x));
  };
  const int four = reinterpret_cast<uintptr_t>(weights + begin) % 16 == 0 ? n / 4 * 4 : 0;
#pragma unroll 8
  for (int i = tid * 4; i < four; i += kThreads * 4) {
    const float4 x = *reinterpret_cast<const float4*>(weights + begin + i);
    *reinterpret_cast<float4*>(row + i) = x;
    look(i, x.x);
    look(i + 1, x.y);
    look(i + 2, x.z);
    look(i + 3, x.w);
  }
  for (int i = four + tid; i < n; i += kThreads) {
    row[i] = weights[begin + i];
    look(i, row[i]);
  }
  // Blocks that lose all their tokens (the stores run beside what follows).
  if (a.lo != nullptr) {
    const int b0 = (now + a.L.b - 1) / a.L.b, b1 = (len + a.L.b - 1) / a.L.b;
    const long long d = a.L.d, from = (base / a.L.b + b0) * d, count = (b1 - b0) * d;
    if ((from | d) % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.lo) | reinterpret_cast<uintptr_t>(a.hi)) & 15) == 0) {
      const float4 none = make_float4(kNothing, kNothing, kNothing, kNothing), no = make_float4(-kNothing, -kNothing, -kNothing, -kNothing);
      for (long long i = at; i < count / 4; i += all) {
        reinterpret_cast<float4*>(a.lo + from)[i] = none;
        reinterpret_cast<float4*>(a.hi + from)[i] = no;
      }
    } else {
      for (long long i = at; i < count; i += all) {
        a.lo[from + i] = kNothing;
        a.hi[from + i] = -kNothing;
      }
    }
  }
  sh.hist[0][tid] = sh.hist[1][tid] = 0;
  if (tid == 0) sh.listed = 0;
  top = __reduce_max_sync(kFull, top);
  if (lane == 0) sh.warp_top[warp] = top;
  __syncthreads();
  top = __reduce_max_sync(kFull, sh.warp_top[lane]);
  if (tid == 0) sh.top = top;
  cluster.sync();
  for (int p = 0; p < parts; ++p) top = max(top, *cluster.map_shared_rank(&sh.top, p));

  // ---- the threshold: `take` tokens whose key is `limit` stay, and all above
  uint32_t limit = 0;
  int take = a.keep - a.first - a.last;
  const bool none = take == 0;  // nothing unprotected stays
  int turn = 0;
  // The thread's bin, over the cluster; the one that reaches the goal is told to all, and the goal left in it.
  auto choose = [&](int& goal) {
    cluster.sync();
    sh.hist[turn ^ 1][tid] = 0;  // (read by siblings before the last meeting)
    int count = 0;
    for (int p = 0; p < parts; ++p) count += cluster.map_shared_rank(sh.hist[turn], p)[tid];
    int total;
    const int before = scan_add<int>(count, sh.warp_sums, total);
    if (before < goal && before + count >= goal) {
      sh.bin = tid;
      sh.above = before;
      sh.crowd = count;
    }
    __syncthreads();
    goal -= sh.above;
    turn ^= 1;
  };
  // Zeros, the weights of tokens that nothing has seen, have a bin of their own before the last, the negative ones'.
  constexpr uint32_t kZero = 0x80000000u;
  auto bin_of = [&](uint32_t key) {
    return key > kZero ? static_cast<int>(min((top - key) >> kBinShift, static_cast<uint32_t>(kBins - 3)))
                       : key == kZero ? kBins - 2 : kBins - 1;
  };
  auto middle = [&](auto f) {
    const int i1 = min(n, hi - begin);
    for (int i = max(0, lo - begin) + tid; i < i1; i += kThreads) f(i, weight_key(row[i]));
  };
  bool found = none;
  if (!none) {
    int goal = take;
    middle([&](int, uint32_t key) { atomicAdd(&sh.hist[turn][bin_of(key)], 1); });
    choose(goal);
    const int bin = sh.bin, crowd = sh.crowd;
    if (bin == kBins - 2) {
      limit = kZero;
      take = goal;
      found = true;
    } else if (crowd <= kThreads) {
      u64* list = cluster.map_shared_rank(sh.list, 0);
      int* listed = cluster.map_shared_rank(&sh.listed, 0);
      middle([&](int i, uint32_t key) {
        if (bin_of(key) == bin) list[atomicAdd(listed, 1)] = static_cast<u64>(key) << 32 | static_cast<uint32_t>(~(begin + i));
      });
      cluster.sync();
      if (part == 0) {
        u64 x = tid < crowd ? sh.list[tid] : 0;
        x = sort_descending(x, crowd, sh.list);
        __syncthreads();
        sh.list[tid] = x;
        __syncthreads();
        if (tid == goal - 1) {  // the last one that stays, and how many of its weight do
          const uint32_t key = static_cast<uint32_t>(x >> 32);
          int first = tid, l = 0;
          while (l < first) {
            const int mid = (l + first) >> 1;
            if (static_cast<uint32_t>(sh.list[mid] >> 32) > key) l = mid + 1; else first = mid;
          }
          sh.limit = key;
          sh.take = tid - first + 1;
        }
      }
      cluster.sync();
      limit = *cluster.map_shared_rank(&sh.limit, 0);
      take = *cluster.map_shared_rank(&sh.take, 0);
      found = true;
    }
  }
  if (!found) {
    for (int digit = 0; digit < 4; ++digit) {  // 10, 10, 10 and 2 bits
      const int shift = digit == 3 ? 0 : 22 - 10 * digit, bits = digit == 3 ? 2 : 10;
      middle([&](int, uint32_t key) {
        if (digit == 0 || (key >> (shift + bits)) == (limit >> (shift + bits)))
          atomicAdd(&sh.hist[turn][kBins - 1 - static_cast<int>((key >> shift) & ((1u << bits) - 1))], 1);
      });
      choose(take);
      limit |= static_cast<uint32_t>(kBins - 1 - sh.bin) << shift;
      __syncthreads();
    }
  }

  // ---- each warp's stretch: tokens above, and at, the threshold
  const int stretch = (n + 32 * 32 - 1) / (32 * 32) * 32, w0 = min(n, warp * stretch), w1 = min(n, w0 + stretch);
  auto kind = [&](int i) {  // 2: stays, 1: at the threshold
    const int place = begin + i;
    if (place < lo || place >= hi) return 2;
    const uint32_t key = weight_key(row[i]);
    return none ? 0 : key > limit ? 2 : key == limit ? 1 : 0;
  };
  int above = 0, equal = 0;
#pragma unroll 4
  for (int i0 = w0; i0 < w1; i0 += 32) {
    const int k = i0 + lane < w1 ? kind(i0 + lane) : 0;
    const unsigned a2 = __ballot_sync(kFull, k == 2), a1 = __ballot_sync(kFull, k == 1);
    if (lane == 0) sh.kinds[i0 / 32] = make_uint2(a2, a1);
    above += __popc(a2);
    equal += __popc(a1);
  }
  int all_above, all_equal;
  above = scan_add<int>(lane == 0 ? above : 0, sh.warp_sums, all_above);
  equal = scan_add<int>(lane == 0 ? equal : 0, sh.warp_sums, all_equal);
  above = __shfl_sync(kFull, above, 0);
  equal = __shfl_sync(kFull, equal, 0);
  if (tid == 0) sh.count = make_int2(all_above, all_equal);
  cluster.sync();
  for (int p = 0; p < part; ++p) {
    const int2 c = *cluster.map_shared_rank(&sh.count, p);
    above += c.x;
    equal += c.y;
  }
  __syncwarp();
  const unsigned below = (1u << lane) - 1;
  const int chunk_shift = __ffs(a.chunk) - 1;
#pragma unroll 4
  for (int i0 = w0; i0 < w1; i0 += 32) {
    const uint2 kinds = sh.kinds[i0 / 32];
    const int i = i0 + lane, place = begin + i;
    const int e = equal + __popc(kinds.y & below), goal = above + __popc(kinds.x & below) + min(e, take);
    if ((kinds.x >> lane & 1) || ((kinds.y >> lane & 1) && e < take)) {
      kept[goal] = place;
      out[goal] = row[i];
    }
    if ((place & (a.chunk - 1)) == 0 && i < w1 && place <= a.chunk * a.chunks) rank[place >> chunk_shift] = goal;
    above += __popc(kinds.x);
    equal += __popc(kinds.y);
  }
  for (int i = at; i <= a.chunks; i += all)
    if (i * a.chunk >= len) rank[i] = a.keep;
  for (int i = a.keep + at; i < room; i += all) out[i] = 0.f;
  cluster.sync();  // the counts have been read
}

// ---------------------------------------------------------------- the move

template <int BYTES>
struct Piece;
template <>
struct Piece<16> { using type = uint4; };
template <>
struct Piece<4> { using type = uint32_t; };
template <>
struct Piece<2> { using type = unsigned short; };

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

constexpr int kMoveWarps = 28, kSteps = 16;  // warps of a CTA at most, steps of a chunk
static_assert(32 / kEvictSegment * kSteps >= 32, "a chunk is 32 rows at most");
constexpr int kStageBytes = kSteps * 32 * 16;  // a warp's chunk in shared memory

template <int PIECE>
__device__ __forceinline__ void copy_piece(void* to, const void* from) {
  if constexpr (PIECE == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory");
  else if constexpr (PIECE == 4)
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(to)), "l"(from) : "memory");
  else
    *static_cast<unsigned short*>(to) = *static_cast<const unsigned short*>(from);
}

// Least and largest of the values of a piece, NaN where any is: 16-bit ones in pairs.
template <typename T, int PIECE>
struct Bounds {
  static constexpr bool kPairs = sizeof(T) == 2 && PIECE >= 4;
  static constexpr int E = PIECE / static_cast<int>(sizeof(T)), N = kPairs ? E / 2 : E;
  using V = typename std::conditional<!kPairs, float, typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type>::type;
  V low[N], high[N];
  static __device__ __forceinline__ V least(V a, V b) {
    if constexpr (kPairs) return __hmin2_nan(a, b);
    else return min_nan(a, b);
  }
  static __device__ __forceinline__ V most(V a, V b) {
    if constexpr (kPairs) return __hmax2_nan(a, b);
    else return max_nan(a, b);
  }
  static __device__ __forceinline__ V shuffle(V x, int lane) {
    uint32_t u = __shfl_sync(kFull, *reinterpret_cast<const uint32_t*>(&x), lane);
    return *reinterpret_cast<const V*>(&u);
  }
  __device__ __forceinline__ void take(const void* piece, bool first) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      V v;
      if constexpr (kPairs) v = static_cast<const V*>(piece)[i];
      else v = to_f32(static_cast<const T*>(piece)[i]);
      low[i] = first ? v : least(low[i], v);
      high[i] = first ? v : most(high[i], v);
    }
  }
  __device__ __forceinline__ void put(float* lo, float* hi) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (kPairs) {
        lo[2 * i] = to_f32(low[i].x);
        lo[2 * i + 1] = to_f32(low[i].y);
        hi[2 * i] = to_f32(high[i].x);
        hi[2 * i + 1] = to_f32(high[i].y);
      } else {
        lo[i] = low[i];
        hi[i] = high[i];
      }
    }
  }
};

// A chunk on its way: the rows of the pool that the lane's token of it is in and goes to, and its block.
struct Chunk {
  uint32_t source, goal;
  int c, first, count, id, block;
  bool keys, moves, opens, closes;  // of the block's chunks
  int segment;
};
constexpr uint32_t kNoRow = 0xffffffffu;  // its page lies outside the pool

// PIECE: bytes that a lane moves at once. PIECES: of each segment of a row, 0: any
// number. An item is one block of a row (all its chunks in
// order), of K or of V, one segment.
template <typename T, int PIECE, int PIECES>
__global__ void __launch_bounds__(kMoveWarps * 32, 1) evict_move_kernel(const EvictArgs a, int items) {
  using P = typename Piece<PIECE>::type;
  constexpr int E = PIECE / static_cast<int>(sizeof(T));
  extern __shared__ __align__(16) unsigned char stages[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned char* stage = stages + warp * kStageBytes;
  const int rows = a.R * a.L.hkv, per = rows * 2 * a.segments;
  const int pieces = a.L.d / E, ps = a.L.page_size, ppb = a.L.b / ps, row_bytes = pieces * PIECE;
  const int ps_shift = (ps & (ps - 1)) == 0 ? __ffs(ps) - 1 : -1, chunk_shift = __ffs(a.chunk) - 1;
  const int warps = static_cast<int>(gridDim.x) * (static_cast<int>(blockDim.x) >> 5);
  int item = static_cast<int>(blockIdx.x) + warp * static_cast<int>(gridDim.x) - warps;
  // The item's block.
  int id = 0, h = 0, segment = 0, t0 = 0, tokens = 0, next = 0, at_block = 0;
  bool keys = false;
  const int* kept = nullptr;
  const int* table = nullptr;
  // The lane's place in a step: which of the rows at once, which piece.
  int np = PIECES, at_once = PIECES ? 32 / (PIECES ? PIECES : 1) : 0, group = PIECES ? lane / (PIECES ? PIECES : 1) : 0;
  int column = PIECES ? lane % (PIECES ? PIECES : 1) : 0, set = -1;
  auto lanes_of = [&](int seg) {
    if (PIECES || seg == set) return;
    set = seg;
    np = min(kEvictSegment, pieces - seg * kEvictSegment);
    at_once = 32 / np;
    group = lane / np;
    column = lane - group * np;
  };
  // The next chunk that has something to do: its tokens' places.
  auto fetch = [&](Chunk& x) {
    while (next >= t0 + tokens) {
      item += warps;
      if (item >= items) return false;
      const int block = item / per;
      int rest = item - block * per;
      const int line = rest / rows;
      id = rest - line * rows;
      keys = line % 2 == 0;
      segment = line / 2;
      const int r = id / a.L.hkv;
      h = id - r * a.L.hkv;
      tokens = 0;
      next = t0 = block * a.L.b;
      const int b0 = a.L.block_offsets[r];
      if (held_tokens(a, r) <= a.keep) continue;
      kept = a.kept + static_cast<long long>(id) * a.keep;
      const int most = min(a.L.b, a.keep - t0);
      // A full block whose last token stays in place is what it was.
      if (most == a.L.b && kept[t0 + most - 1] == t0 + most - 1) continue;
      tokens = most;
      at_block = b0 + block;
      table = a.L.page_table + static_cast<long long>(b0) * ppb;
    }
    x.first = next;
    x.c = next >> chunk_shift;
    x.count = min(a.chunk, t0 + tokens - next);
    x.id = id;
    x.block = at_block;
    x.segment = segment;
    x.keys = keys;
    x.opens = next == t0;
    next += x.count;
    x.closes = next >= t0 + tokens;
    const int to = x.first + min(lane, x.count - 1), from = kept[to];
    auto place = [&](int token) {
      const int in = ps_shift >= 0 ? token >> ps_shift : token / ps;
      const int page = table[in];
      if (page < 0 || page >= a.pages) {
        report(a.status, kStatusBadBlockId);
        return kNoRow;
      }
      return static_cast<uint32_t>((page * a.L.hkv + h) * ps + (token - in * ps));
    };
    x.source = place(from);
    x.goal = place(to);
    x.moves = __any_sync(kFull, from != to);
    return true;
  };
  auto pool_of = [&](const Chunk& x) {
    return static_cast<unsigned char*>(const_cast<void*>(x.keys ? a.L.k : a.L.v)) + (x.segment * kEvictSegment + column) * PIECE;
  };
  auto load = [&](const Chunk& x) {
    lanes_of(x.segment);
    const unsigned char* pool = pool_of(x);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      if (i * at_once >= x.count) break;
      const int t = i * at_once + group;
      const uint32_t s = __shfl_sync(kFull, x.source, t & 31);
      if ((PIECES || group < at_once) && t < x.count && s != kNoRow)
        copy_piece<PIECE>(stage + (i * 32 + lane) * PIECE, pool + static_cast<unsigned long long>(s) * row_bytes);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  Bounds<T, PIECE> bounds;
  bool started = false;  // the lane has seen a value of the block
  bool ok = true;
  auto store = [&](const Chunk& x) {
    lanes_of(x.segment);
    if (x.moves) {
      int* read = a.read + (static_cast<long long>(x.id) * 2 * a.segments + x.segment * 2 + (x.keys ? 0 : 1)) * a.chunks;
      const int* rank = a.rank + static_cast<long long>(x.id) * (a.chunks + 1);
      // The earlier chunks of kept tokens that lie in this chunk's places.
      const int i0 = rank[x.c], i1 = min(rank[x.c + 1], x.first);
      __syncwarp();  // all lanes have read the chunk before the release
      if (lane == 0) asm volatile("st.release.gpu.global.s32 [%0], 1;" ::"l"(read + x.c) : "memory");
      if (i0 < i1) {
        const int* flag = read + min((i0 >> chunk_shift) + lane, (i1 - 1) >> chunk_shift);
        auto seen = [&]() {
          int f;
          asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(f) : "l"(flag) : "memory");
          return f != 0;
        };
        // (A chunk that does not move reads its own places alone: nobody waits for it.)
        if (!__all_sync(kFull, seen())) {
          const unsigned long long began = global_ns();
          while (!__all_sync(kFull, seen())) {
            if (__any_sync(kFull, global_ns() - began > c_wait_ns)) {
              report(a.status, kStatusWaitTimeout);
              ok = false;
              return;
            }
          }
        }
        __syncwarp();
      }
    }
    const bool bounded = x.keys && a.lo != nullptr;
    if (x.opens) started = false;
    unsigned char* pool = pool_of(x);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      if (i * at_once >= x.count) break;
      const int t = i * at_once + group;
      const uint32_t s = __shfl_sync(kFull, x.source, t & 31), g = __shfl_sync(kFull, x.goal, t & 31);
      if ((!PIECES && group >= at_once) || t >= x.count || s == kNoRow || g == kNoRow) continue;
      const P v = *reinterpret_cast<const P*>(stage + (i * 32 + lane) * PIECE);
      if (s != g) *reinterpret_cast<P*>(pool + static_cast<unsigned long long>(g) * row_bytes) = v;
      if (bounded) {
        bounds.take(&v, !started);
        started = true;
      }
    }
    if (bounded && x.closes) {
      // Lanes of the same pieces: those without a value (fewer rows than lanes) take another's.
      const unsigned have = __ballot_sync(kFull, started);
      unsigned peers = 0;
      for (int g = 0; g < at_once; ++g) peers |= 1u << (column + g * np);
      peers &= have;
      for (int g = 0; g < at_once; ++g) {
        const int other = (column + g * np) & 31;
        Bounds<T, PIECE> y = bounds;
#pragma unroll
        for (int i = 0; i < Bounds<T, PIECE>::N; ++i) {
          y.low[i] = Bounds<T, PIECE>::shuffle(bounds.low[i], other);
          y.high[i] = Bounds<T, PIECE>::shuffle(bounds.high[i], other);
        }
        if (group == 0 && g > 0 && (peers >> other & 1)) {
#pragma unroll
          for (int i = 0; i < Bounds<T, PIECE>::N; ++i) {
            bounds.low[i] = started ? Bounds<T, PIECE>::least(bounds.low[i], y.low[i]) : y.low[i];
            bounds.high[i] = started ? Bounds<T, PIECE>::most(bounds.high[i], y.high[i]) : y.high[i];
          }
          started = true;
        }
      }
      if (group == 0 && started) {
        const int hh = x.id % a.L.hkv;
        const long long at = (hh * (a.slots / a.L.b) + x.block) * static_cast<long long>(a.L.d) + (x.segment * kEvictSegment + column) * E;
        bounds.put(a.lo + at, a.hi + at);
      }
    }
  };
  Chunk x[2];
  bool more = fetch(x[0]);
  while (more) {  // two states by turns: the next chunk's places are looked up while one's rows are on their way
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (!more) break;
      load(x[s]);
      more = fetch(x[s ^ 1]);
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      __syncwarp();
      store(x[s]);
      __syncwarp();
      if (!ok) more = false;
    }
  }
}

template <typename T, int PIECE, int PIECES>
int launch_pieces(const EvictArgs& a, int sms, cudaStream_t stream) {
  EvictArgs args = a;
  const long long all = static_cast<long long>((a.keep + a.L.b - 1) / a.L.b) * a.R * a.L.hkv * 2 * a.segments;
  if (all > 0x7fffffff - sms * kMoveWarps) return static_cast<int>(cudaErrorInvalidValue);
  int items = static_cast<int>(all);
  auto kern = evict_move_kernel<T, PIECE, PIECES>;
  const int rc = static_cast<int>(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMoveWarps * kStageBytes));
  if (rc) return rc;
  const int grid = items < sms ? items : sms;  // all of them resident: they wait for one another
  const int each = (items + grid - 1) / grid, warps = each < kMoveWarps ? each : kMoveWarps;
  void* params[] = {&args, &items};
  return static_cast<int>(cudaLaunchCooperativeKernel(reinterpret_cast<const void*>(kern), dim3(grid), dim3(warps * 32), params,
                                                      static_cast<size_t>(warps) * kStageBytes, stream));
}

template <typename T, int PIECE>
int launch_move(const EvictArgs& a, int sms, cudaStream_t stream) {
  if (PIECE == 16) {
    const int pieces = a.L.d * static_cast<int>(sizeof(T)) / 16;
    if (pieces == 8) return launch_pieces<T, PIECE, PIECE == 16 ? 8 : 0>(a, sms, stream);
    if (pieces % 16 == 0) return launch_pieces<T, PIECE, PIECE == 16 ? 16 : 0>(a, sms, stream);
  }
  return launch_pieces<T, PIECE, 0>(a, sms, stream);
}

}  // namespace

int launch_evict_select(const EvictArgs& a, int sms, cudaStream_t stream) {
  const long long rows = static_cast<long long>(a.R) * a.L.hkv;
  // CTAs of a row: as many as its tokens need, more while they find SMs and
  // 16 K tokens each. A request of two heads cut to 2 K tokens takes 43.8 us from
  // 32,000 by the two CTAs of this rule (by one 64, four 35, eight 31), 44.5 from
  // 16,000 by its one (by two 34.4, four 30.2).
  int parts = 1;
  while (parts * kEvictSlice < a.longest) parts *= 2;
  while (parts < kEvictCluster && rows * parts * 2 <= sms && a.longest / parts > 16384) parts *= 2;
  if (rows * parts > 0x7fffffff) return static_cast<int>(cudaErrorInvalidValue);
  const int bytes = static_cast<int>(sizeof(float)) * (((a.longest + parts - 1) / parts + 31) / 32 * 32);
  auto kern = evict_select_kernel;
  int rc = static_cast<int>(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kEvictSlice * 4));
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * parts));
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

int launch_evict_move(const EvictArgs& a, int kv_dtype, int piece, int sms, cudaStream_t stream) {
  if (kv_dtype == kF32) return piece == 16 ? launch_move<float, 16>(a, sms, stream) : launch_move<float, 4>(a, sms, stream);
  if (kv_dtype == kBF16)
    return piece == 16  ? launch_move<__nv_bfloat16, 16>(a, sms, stream)
           : piece == 4 ? launch_move<__nv_bfloat16, 4>(a, sms, stream)
                        : launch_move<__nv_bfloat16, 2>(a, sms, stream);
  return piece == 16  ? launch_move<__half, 16>(a, sms, stream)
         : piece == 4 ? launch_move<__half, 4>(a, sms, stream)
                      : launch_move<__half, 2>(a, sms, stream);
}

}  // namespace stk
