// Eviction from a paged cache: of each request's KV head the tokens of the
// largest weights stay (ties to the lower place; the first and last ones are
// protected), in their order, at the front of the request's own pages.
//
// Selection: a row (request, KV head) lies in the shared memory of a cluster
// of up to eight CTAs, read once. The threshold is found digit by digit (11, 11
// and 10 bits of the weights' order keys), the histograms summed over the
// cluster; then every warp counts and writes its stretch in order: IDs, weights
// and, for the move, how many kept tokens lie before each chunk.
//
// Move: kept token i goes to place i <= its own. Moving in place saves half the
// bytes of a way through a copy, but a place may be overwritten only after it
// has been read. A warp reads a chunk into registers, announces that, waits for
// the (at most two) earlier chunks that read the places it writes, and writes.
// The warps of a co-resident grid take chunks in ascending order, so each waits
// for earlier ones only and some warp can always go on. A block's key bounds are
// taken on the way by the warp that moves its keys.

#include <cooperative_groups.h>

#include <type_traits>

#include "evict.cuh"

namespace stk {

int set_wait_limit_evict(unsigned long long ns) { return set_wait_limit_this_unit(ns); }

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 1024, kBins = 2048;
constexpr float kNothing = 1e30f;  // lo, and minus hi, of a block without tokens

// Weights in ascending order, NaN above all, zeros of either sign alike.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x);
  if (x != x) return 0xffffffffu;
  if (x == 0.f) return 0x80000000u;
  return u ^ (u >> 31 ? 0xffffffffu : 0x80000000u);
}

// Tokens of request r, at most as many as its blocks hold.
__device__ __forceinline__ int held_tokens(const EvictArgs& a, int r) {
  const int n = a.lengths[r], room = request_blocks(a.L, r) * a.L.b;
  if (n < 0 || n > room) report(a.status, kStatusBadLength);
  return max(0, min(n, min(room, a.longest)));
}

// Exclusive prefix sums of v over the CTA's threads, and its total. Two barriers.
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(kFull, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  int s = warp_sums[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(kFull, s, o);
    if (lane >= o) s += y;
  }
  total = __shfl_sync(kFull, s, 31);
  const int before = warp ? __shfl_sync(kFull, s, warp - 1) : 0;
  return before + x - v;
}

struct SelectShared {
  int hist[2][kBins];  // of two digits by turns: a sibling may still read the last one's
  int warp_sums[32];
  int2 count;          // of the CTA: tokens above the threshold (or protected), tokens at it
  int digit, above, inside;
};

__global__ void __launch_bounds__(kThreads, 1) evict_select_kernel(const EvictArgs a) {
  extern __shared__ float row[];
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
  for (int i = tid; i < n; i += kThreads) row[i] = weights[begin + i];
  for (int i = tid; i < kBins; i += kThreads) sh.hist[0][i] = 0;
  __syncthreads();

  // ---- the threshold: `take` tokens whose key is `limit` stay, and all above
  const int lo = a.first, hi = len - a.last;  // the others of the row are protected
  uint32_t limit = 0;
  int take = a.keep - a.first - a.last;
  bool found = take == 0;  // (then nothing unprotected stays)
  if (found) limit = 0xffffffffu;
  for (int digit = 0; digit < 3; ++digit) {
    const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0, bits = digit == 2 ? 10 : 11;
    int* hist = sh.hist[digit & 1];
    if (!found) {
      for (int i = tid; i < n; i += kThreads) {
        const uint32_t key = order_key(row[i]);
        const bool in = begin + i >= lo && begin + i < hi && (digit == 0 || (key >> (shift + bits)) == (limit >> (shift + bits)));
        if (in) atomicAdd(&hist[(key >> shift) & ((1u << bits) - 1)], 1);
      }
    }
    cluster.sync();
    if (digit < 2)
      for (int i = tid; i < kBins; i += kThreads) sh.hist[(digit & 1) ^ 1][i] = 0;  // (read by siblings before the last sync)
    // Two bins per thread, the highest first.
    const int top = kBins - 1 - 2 * tid;
    int c0 = 0, c1 = 0;
    for (int p = 0; p < parts; ++p) {
      const int* other = cluster.map_shared_rank(hist, p);
      c0 += other[top];
      c1 += other[top - 1];
    }
    int total;
    const int before = block_scan(c0 + c1, sh.warp_sums, total);
    if (!found) {
      if (before < take && before + c0 >= take) {
        sh.digit = top;
        sh.above = before;
        sh.inside = c0;
      } else if (before + c0 < take && before + c0 + c1 >= take) {
        sh.digit = top - 1;
        sh.above = before + c0;
        sh.inside = c1;
      }
    }
    __syncthreads();
    if (!found) {
      limit |= static_cast<uint32_t>(sh.digit) << shift;
      take -= sh.above;
    }
    __syncthreads();
  }

  // ---- each warp's stretch: tokens above, and at, the threshold
  const int stretch = (n + 32 * 32 - 1) / (32 * 32) * 32, w0 = min(n, warp * stretch), w1 = min(n, w0 + stretch);
  auto kind = [&](int i) {  // 2: stays, 1: at the threshold
    const int place = begin + i;
    if (place < lo || place >= hi) return 2;
    const uint32_t key = order_key(row[i]);
    return found ? 0 : key > limit ? 2 : key == limit ? 1 : 0;
  };
  int above = 0, equal = 0;
  for (int i0 = w0; i0 < w1; i0 += 32) {
    const int k = i0 + lane < w1 ? kind(i0 + lane) : 0;
    above += __popc(__ballot_sync(kFull, k == 2));
    equal += __popc(__ballot_sync(kFull, k == 1));
  }
  int all_above, all_equal;
  above = block_scan(lane == 0 ? above : 0, sh.warp_sums, all_above);
  equal = block_scan(lane == 0 ? equal : 0, sh.warp_sums, all_equal);
  above = __shfl_sync(kFull, above, 0);
  equal = __shfl_sync(kFull, equal, 0);
  if (tid == 0) sh.count = make_int2(all_above, all_equal);
  cluster.sync();
  for (int p = 0; p < part; ++p) {
    const int2 c = *cluster.map_shared_rank(&sh.count, p);
    above += c.x;
    equal += c.y;
  }
  for (int i0 = w0; i0 < w1; i0 += 32) {
    const int i = i0 + lane, place = begin + i;
    const int k = i < w1 ? kind(i) : 0;
    const unsigned a2 = __ballot_sync(kFull, k == 2), a1 = __ballot_sync(kFull, k == 1), below = (1u << lane) - 1;
    const int e = equal + __popc(a1 & below), goal = above + __popc(a2 & below) + min(e, take);
    if (k == 2 || (k == 1 && e < take)) {
      kept[goal] = place;
      out[goal] = row[i];
    }
    if (i < w1 && place % a.chunk == 0 && place / a.chunk <= a.chunks) rank[place / a.chunk] = goal;
    above += __popc(a2);
    equal += __popc(a1);
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

constexpr int kMoveThreads = 256, kSteps = 16;

// PIECE: bytes that a lane moves at once. An item is one block of a row (all
// its chunks in order), of K or of V, one segment of up to 32 pieces.
template <typename T, int PIECE>
__global__ void __launch_bounds__(kMoveThreads, 2) evict_move_kernel(const EvictArgs a, long long items) {
  using P = typename Piece<PIECE>::type;
  constexpr int E = PIECE / static_cast<int>(sizeof(T));
  const int lane = threadIdx.x & 31;
  const int rows = a.R * a.L.hkv, per = rows * 2 * a.segments;
  const int pieces = a.L.d / E, ps = a.L.page_size, chunks_per_block = a.L.b / a.chunk;
  bool ok = true;
  const long long warps = static_cast<long long>(gridDim.x) * (kMoveThreads / 32);
  for (long long item = blockIdx.x * (kMoveThreads / 32) + (threadIdx.x >> 5); item < items && ok; item += warps) {
    const int block = static_cast<int>(item / per);
    int rest = static_cast<int>(item - static_cast<long long>(block) * per);
    const int id = rest % rows;
    rest /= rows;
    const bool keys = rest % 2 == 0;
    const int segment = rest / 2, r = id / a.L.hkv, h = id - r * a.L.hkv;
    const int len = held_tokens(a, r);
    if (len <= a.keep || block * a.L.b >= len) continue;
    const int now = a.keep, b0 = a.L.block_offsets[r], t0 = block * a.L.b;
    const int p0 = segment * 32, np = min(32, pieces - p0);  // the segment's pieces
    const int at_once = 32 / np, group = lane / np, column = lane - group * np;
    const bool active = group < at_once;
    const bool bounds = keys && a.lo != nullptr;
    const long long bound_at = (h * (a.slots / a.L.b) + b0 + block) * static_cast<long long>(a.L.d) + (p0 + column) * E;
    if (t0 >= now) {  // a block that holds nothing any more
      if (bounds && group == 0)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          a.lo[bound_at + e] = kNothing;
          a.hi[bound_at + e] = -kNothing;
        }
      continue;
    }
    const int* kept = a.kept + static_cast<long long>(id) * a.keep;
    const int tokens = min(a.L.b, now - t0);
    // A full block whose last token stays in place is what it was.
    if (tokens == a.L.b && kept[t0 + tokens - 1] == t0 + tokens - 1) continue;
    T* pool = static_cast<T*>(const_cast<void*>(keys ? a.L.k : a.L.v));
    const int* table = a.L.page_table + static_cast<long long>(b0) * (a.L.b / ps);
    const int* rank = a.rank + static_cast<long long>(id) * (a.chunks + 1);
    int* read = a.read + (static_cast<long long>(id) * 2 * a.segments + segment * 2 + (keys ? 0 : 1)) * a.chunks;
    float low[E], high[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      low[e] = __int_as_float(0x7f800000);
      high[e] = -low[e];
    }
    for (int c = t0 / a.chunk; c * a.chunk < t0 + tokens && ok; ++c) {
      const int first = c * a.chunk, count = min(a.chunk, t0 + tokens - first);
      // The lane's token of the chunk: where it is, and where it goes.
      const int to = first + min(lane, count - 1), from = kept[to];
      auto place = [&](int token) {
        int page = table[token / ps];
        if (page < 0 || page >= a.pages) {
          report(a.status, kStatusBadBlockId);
          page = -1;
        }
        return page < 0 ? -1ll : (static_cast<long long>(page) * a.L.hkv + h) * ps + token % ps;
      };
      const long long source = place(from), goal = place(to);
      const bool moves = __any_sync(kFull, from != to);
      P x[kSteps];
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const int t = i * at_once + group;
        const long long s = __shfl_sync(kFull, source, min(t, 31));
        if (active && t < count && s >= 0) x[i] = *reinterpret_cast<const P*>(pool + s * a.L.d + (p0 + column) * E);
      }
      if (moves) {
        __threadfence();  // the chunk has been read before this is seen
        __syncwarp();
        if (lane == 0) *reinterpret_cast<volatile int*>(read + c) = 1;
        // The earlier chunks of kept tokens that lie in this chunk's places.
        const int i0 = rank[c], i1 = min(rank[c + 1], first);
        if (i0 < i1) {
          const int c0 = i0 / a.chunk, c1 = (i1 - 1) / a.chunk;
          const volatile int* flag = read + min(c0 + lane, c1);
          const unsigned long long began = global_ns();
          // (A chunk that does not move reads its own places alone: nobody waits for it.)
          while (!__all_sync(kFull, *flag != 0)) {
            if (global_ns() - began > c_wait_ns) {
              report(a.status, kStatusWaitTimeout);
              ok = false;
            }
            if (__any_sync(kFull, !ok)) {
              ok = false;
              break;
            }
          }
          __threadfence();
        }
      }
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const int t = i * at_once + group;
        const long long s = __shfl_sync(kFull, source, min(t, 31)), g = __shfl_sync(kFull, goal, min(t, 31));
        if (!active || t >= count || s < 0 || g < 0 || !ok) continue;
        if (s != g) *reinterpret_cast<P*>(pool + g * a.L.d + (p0 + column) * E) = x[i];
        if (bounds) {
          const T* v = reinterpret_cast<const T*>(&x[i]);
#pragma unroll
          for (int e = 0; e < E; ++e) {
            low[e] = min_nan(low[e], to_f32(v[e]));
            high[e] = max_nan(high[e], to_f32(v[e]));
          }
        }
      }
    }
    if (bounds && ok) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float l = low[e], u = high[e];
        for (int g = 1; g < at_once; ++g) {
          l = min_nan(l, __shfl_sync(kFull, low[e], (column + g * np) & 31));
          u = max_nan(u, __shfl_sync(kFull, high[e], (column + g * np) & 31));
        }
        if (group == 0) {
          a.lo[bound_at + e] = l;
          a.hi[bound_at + e] = u;
        }
      }
    }
  }
}

template <typename T, int PIECE>
int launch_move(const EvictArgs& a, int sms, cudaStream_t stream) {
  EvictArgs args = a;
  long long items = static_cast<long long>((a.longest + a.L.b - 1) / a.L.b) * a.R * a.L.hkv * 2 * a.segments;
  if (static_cast<long long>(a.R) * a.L.hkv * 2 * a.segments > 0x7fffffff) return static_cast<int>(cudaErrorInvalidValue);
  auto kern = evict_move_kernel<T, PIECE>;
  const long long ctas = (items + kMoveThreads / 32 - 1) / (kMoveThreads / 32);
  const int grid = static_cast<int>(ctas < 2ll * sms ? ctas : 2ll * sms);  // all of them resident: they wait for one another
  void* params[] = {&args, &items};
  return static_cast<int>(cudaLaunchCooperativeKernel(reinterpret_cast<const void*>(kern), dim3(grid), dim3(kMoveThreads), params, 0, stream));
}

}  // namespace

int launch_evict_select(const EvictArgs& a, int sms, cudaStream_t stream) {
  const long long rows = static_cast<long long>(a.R) * a.L.hkv;
  // CTAs of a row: as many as its tokens need, more while they find SMs and a
  // few thousand tokens each.
  int parts = 1;
  while (parts * kEvictSlice < a.longest) parts *= 2;
  while (parts < kEvictCluster && rows * parts * 2 <= sms && a.longest / parts > 4096) parts *= 2;
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
