// Arguments of eviction from a paged cache: which tokens stay, and their move
// to the front of the requests' pages.
#pragma once

#include "paged_ops.cuh"

namespace stk {

struct EvictArgs {
  KVLayout L;
  int pages, R;
  const int* lengths;    // [R] tokens in the cache
  int keep, first, last; // tokens that stay at most, protected at both ends
  int longest;           // bound on a request's tokens
  long long slots;       // token slots of all blocks
  const float* weights;  // [hkv, slots]
  float* weights_out;
  float* lo;             // [hkv, slots / b, d] or null
  float* hi;
  int* kept;             // [R, hkv, keep]
  int* lengths_out;      // [R]
  // Between the two kernels: tokens are moved in chunks, each announced once it
  // has been read.
  int chunk, chunks;     // tokens of a chunk (a power of two that divides b), chunks of `keep` tokens
  int segments;          // parts of a row (of kEvictSegment pieces) that are moved apart
  int* rank;             // [R * hkv, chunks + 1] kept tokens before each chunk's first place
  int* read;             // [R * hkv, 2 * segments, chunks] flags
  int* status;
};

constexpr int kEvictCluster = 8;        // CTAs that share a row at most
constexpr int kEvictSlice = 49152;      // its tokens that one of them holds in shared memory
constexpr int kEvictSegment = 16;       // pieces of a row that are moved together: a chunk of 32 rows in 16 steps of a warp
constexpr int kEvictMost = kEvictCluster * kEvictSlice;

// Bytes of the pieces that rows of the pools are moved in.
inline int evict_piece(int kv_dtype, int d, const void* k, const void* v) {
  const int size = kv_dtype == kF32 ? 4 : 2;
  const uintptr_t any = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | static_cast<uintptr_t>(d * size);
  return any % 16 == 0 ? 16 : any % 4 == 0 ? 4 : 2;
}

// Tokens of a chunk: one to a lane, if they divide the block.
inline void evict_plan(EvictArgs& a, int kv_dtype, int piece) {
  const int row = a.L.d * (kv_dtype == kF32 ? 4 : 2) / piece;
  a.segments = (row + kEvictSegment - 1) / kEvictSegment;
  a.chunk = 1;
  while (a.chunk < 32 && a.L.b % (2 * a.chunk) == 0) a.chunk *= 2;
  a.chunks = a.keep / a.chunk + (a.keep % a.chunk != 0);
}

int launch_evict_select(const EvictArgs& a, int sms, cudaStream_t stream);
int launch_evict_move(const EvictArgs& a, int kv_dtype, int piece, int sms, cudaStream_t stream);
int set_wait_limit_evict(unsigned long long ns);

}  // namespace stk
