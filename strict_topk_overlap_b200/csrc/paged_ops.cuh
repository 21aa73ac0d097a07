// Argument structs and device helpers shared by the paged token append and
// the dense paged attention kernels.
//
// New tokens of a call are packed request after request: request r owns
// tokens token_offsets[r] .. token_offsets[r + 1] (without token_offsets,
// one token each). A token's query heads of one KV head are G consecutive
// "rows"; request r has n_r * G rows per KV head, row = token * G + head.
// Tokens from token_offsets[R] on (padding, as a captured graph has) belong to
// no request: they are the tokens of a request R that holds nothing.
#pragma once

#include "internal.cuh"

namespace stk {

// Status codes of these kernels (see common.cuh for the others).
constexpr int kStatusBadPosition = 4;  // a rotary position outside the table
constexpr int kStatusBadLength = 5;    // a length outside the request's blocks

struct AppendArgs {
  KVLayout L;
  int pages;  // pages in the pool
  int R, T, hq;
  const void* k;  // [T, hkv, d], element strides below
  const void* v;
  const void* q;  // [T, hq, d] or null
  long long k_ts, k_hs, v_ts, v_hs, q_ts, q_hs;
  void* q_out;               // [T, hq, d]
  const int* lengths;        // [R] tokens before the call
  const int* token_offsets;  // [R + 1] or null
  const int* positions;      // [axes, T] or null (lengths[r] + i)
  const float* cos;          // [max_position, pairs] or null (no rotation)
  const float* sin;
  int pairs, max_position, interleaved, axes;
  const unsigned char* axis;  // [pairs] or null
  float* lo;                  // [hkv, total, d] or null
  float* hi;
  int total;
  int* status;
};

struct PagedAttnArgs {
  KVLayout L;
  int pages;
  int R, T, hq, G, d;
  const void* q;
  long long q_ts, q_hs;  // element strides of a token and of a head
  void* out;             // [T, hq, d]
  float* lse;            // [T, hq] or null
  const int* lengths;    // [R] tokens in the cache, the new ones included
  const int* token_offsets;
  const int* kv_lo;  // [T] or null: 0
  const int* kv_hi;  // [T] or null: causal
  const float* slopes;
  float softcap, scale;
  int span_lo, span_hi;  // only keys in [span_lo, span_hi)
  int shared;            // 1: every token reads the pages of request 0
  int nsplit;            // parts of a tile's key range
  int chained;           // launched while the call's first phase still runs: ends after it
  float2* part_ml;       // [nsplit, T * hq] (m, l) of each part; null: the output is written
  float* part_o;         // [nsplit, T * hq, d] unnormalised
  int* status;
};

// Request of slot `slot` when request r's slots start at offs[r] * mul / div + r * add
// (monotone in r): the last r whose first slot is <= slot. One warp; every
// lane returns it.
__device__ __forceinline__ int request_of_slot(const int* offs, int R, int mul, int div, int add, int slot, int lane) {
  int count = 0;
  for (int r0 = 0; r0 < R; r0 += 32) {
    const int r = r0 + lane;
    const bool le = r < R && static_cast<int>(static_cast<long long>(offs[r]) * mul / div) + r * add <= slot;
    const int c = __popc(__ballot_sync(kFull, le));
    count += c;
    if (c < 32) break;
  }
  return max(count - 1, 0);
}

// First packed token and number of new tokens of request r < R, or of the
// padding, r = R. Offsets that do not start at 0, run backwards or go past the
// T tokens are cut to them and reported.
__device__ __forceinline__ int2 new_tokens(const int* offs, int r, int R, int T, int* status) {
  if (offs == nullptr) return make_int2(r, 1);
  const int a = offs[r], b = r < R ? offs[r + 1] : max(a, T);
  if (r < R && (a < 0 || b < a || b > T || (r == 0 && a > 0))) report(status, kStatusShapeOverflow);
  const int first = min(max(a, 0), T);
  return make_int2(first, max(0, min(b, T) - first));
}

// The last request that starts at or before a packed token, R for padding.
__device__ __forceinline__ int request_of_token(const int* offs, int R, int token) {
  if (offs == nullptr) return token;
  int r = 0, end = R + 1;
  while (end - r > 1) {
    const int mid = (r + end) >> 1;
    if (offs[mid] <= token) r = mid; else end = mid;
  }
  return r;
}

// Rows [row0, row0 + rows) of request r: n new tokens from packed token t0
// on, `len` tokens in the cache. Behind a shared prefix all T tokens are the
// rows of one request and r, len are those of its page table, request 0.
struct RowTile {
  int r, row0, rows, t0, n, len;
};

// Tokens of request r in the cache, at most as many as its blocks hold.
__device__ __forceinline__ int cached_tokens(const PagedAttnArgs& a, int r, int n) {
  if (r >= a.R) return 0;  // padding
  const int len = a.lengths[r], room = request_blocks(a.L, r) * a.L.b;
  if (n > 0 && (len > room || len < n)) report(a.status, kStatusBadLength);
  return min(len, room);
}

// Row tile of slot `slot` for tiles of M rows. Request r's ceil(n_r G / M)
// tiles start at slot floor(offs[r] G / M) + r, which leaves room for them
// whatever the lengths; slots without a tile get rows = 0. Warp-converged.
template <int M>
__device__ __forceinline__ RowTile row_tile(const PagedAttnArgs& a, int slot, int lane) {
  RowTile t;
  int f = slot;
  if (a.shared) {
    t.r = t.t0 = 0;
    t.n = a.T;
  } else if (a.token_offsets == nullptr) {
    const int per = (a.G + M - 1) / M;
    t.r = slot / per;
    f = slot - t.r * per;
    t.t0 = t.r;
    t.n = 1;
  } else {
    t.r = request_of_slot(a.token_offsets, a.R + 1, a.G, M, 1, slot, lane);
    const int2 tn = new_tokens(a.token_offsets, t.r, a.R, a.T, a.status);
    t.t0 = tn.x;
    t.n = tn.y;
    f = slot - static_cast<int>(static_cast<long long>(t.t0) * a.G / M) - t.r;
  }
  t.len = a.shared ? request_blocks(a.L, 0) * a.L.b : cached_tokens(a, t.r, t.n);  // loaded beside the offsets
  t.row0 = max(f, 0) * M;
  t.rows = f < 0 ? 0 : max(0, min(M, t.n * a.G - t.row0));
  return t;
}

inline int row_tile_slots(int R, int T, int G, bool offsets, bool shared, int M) {
  if (shared) return static_cast<int>((static_cast<long long>(T) * G + M - 1) / M);
  return offsets ? static_cast<int>(static_cast<long long>(T) * G / M) + R + 1 : R * ((G + M - 1) / M);
}

// Keys lo <= j < hi that token i of a tile's request sees inside the call's
// span, and the token's place in its own request.
struct RowKeys {
  int lo, hi, pos;
};

__device__ __forceinline__ int2 given_keys(const PagedAttnArgs& a, int token) {
  return make_int2(a.kv_lo ? a.kv_lo[token] : 0, a.kv_hi ? a.kv_hi[token] : 0);
}

// `given`: given_keys of the token, loaded ahead of their use.
__device__ __forceinline__ RowKeys row_keys(const PagedAttnArgs& a, const RowTile& t, int i, int2 given) {
  const int token = t.t0 + i;
  RowKeys k;
  int len = t.len;
  if (!a.shared) {
    k.pos = t.len - t.n + i;
  } else {
    const int r = request_of_token(a.token_offsets, a.R, token);
    const int2 tn = new_tokens(a.token_offsets, r, a.R, a.T, a.status);
    len = cached_tokens(a, r, tn.y);
    k.pos = len - (tn.x + tn.y - token);
  }
  k.lo = max(given.x, a.span_lo);
  k.hi = min(min(a.kv_hi ? given.y : k.pos + 1, min(len, t.len)), a.span_hi);
  k.hi = max(k.lo, k.hi);
  return k;
}

__device__ __forceinline__ RowKeys row_keys(const PagedAttnArgs& a, const RowTile& t, int i) {
  return row_keys(a, t, i, given_keys(a, t.t0 + i));
}

// Page of key token `j` of request `rp`, or -1 (reported) when its table
// entry lies outside the pool.
__device__ __forceinline__ int page_of(const PagedAttnArgs& a, int rp, int j) {
  const long long entry = static_cast<long long>(a.L.block_offsets[rp]) * (a.L.b / a.L.page_size) + j / a.L.page_size;
  const int page = a.L.page_table[entry];
  if (page < 0 || page >= a.pages) {
    report(a.status, kStatusBadBlockId);
    return -1;
  }
  return page;
}

// The maximum of a softmax state as it is handed on: -inf says that the row
// saw no key. Scores that are all NaN leave the running maximum there too
// (fmaxf drops them) with a sum of NaN; such a state must reach the output.
__device__ __forceinline__ float state_max(float m, float l) { return m == neg_inf() && l != l ? 0.f : m; }

int launch_append_tokens(const AppendArgs& a, int kv_dtype, int sms, cudaStream_t stream);
int launch_rows_attn(const PagedAttnArgs& a, int kv_dtype, cudaStream_t stream);
// Whether the tensor-core kernel takes these types, sizes and addresses.
bool prompt_attn_takes(int kv_dtype, int d, int page_size, const void* k, const void* v, const void* q, long long q_ts,
                       long long q_hs, const void* out);
// Rows of its CTAs, and how many of them an SM holds.
inline int prompt_tile_rows(int d) { return d == 64 ? 128 : 256; }
inline int prompt_ctas_per_sm(int d) { return d == 64 ? 2 : 1; }
int launch_prompt_attn(const PagedAttnArgs& a, int kv_dtype, cudaStream_t stream);
int set_wait_limit_prompt(unsigned long long ns);

// Few rows per KV head (see token_attn.cu): `streams` warps (a multiple of
// 4) share the batch's units evenly; warp w's state of KV head h of request r
// is partial w + r * hkv + h, most_rows rows each. Writes the units before
// each request to prefix [requests + 1].
bool token_attn_takes(int kv_dtype, int d, int page_size, int R, const void* k, const void* v, const void* q,
                      long long q_ts, long long q_hs);
int launch_token_attn(const PagedAttnArgs& a, int kv_dtype, int streams, int most_rows, int* prefix, cudaStream_t stream);
int set_wait_limit_token(unsigned long long ns);

// One set of partial softmax states to be joined. Without prefix, part s of
// row `row` is at ml[s * rows + row], o[(s * rows + row) * d]; with it, the
// parts are those that token_attn wrote.
struct PartSource {
  const float2* ml;
  const float* o;
  int parts;
  const int* prefix;
  int streams, most_rows, requests, shared;
};

struct JoinArgs {
  PartSource src[2];
  int nsrc, rows, d, dtype;
  int hq, G;
  const int* token_offsets;
  void* out;
  float* lse;
  // Behind a shared prefix: request 0's blocks have to hold it.
  const int* block_offsets;  // null without one
  int block, prefix;
  int* status;
};

int launch_join(const JoinArgs& a, int sms, cudaStream_t stream);

}  // namespace stk
