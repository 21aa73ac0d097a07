// Arguments of the kernels that add up the attention weight each cached key
// receives: weights[h, j] += sum over the new tokens t that see key j and the
// G query heads of KV head h of exp(s - lse[t]).
#pragma once

#include "paged_ops.cuh"

namespace stk {

struct WeighArgs {
  PagedAttnArgs a;     // queries, cache, masks and score options (out, parts and the shared prefix unused)
  const float* lse;    // [T, hq] log-sum-exps of the rows' scores
  float* weights;      // [hkv, slots]
  long long slots;     // token slots of all blocks
  int most;            // bound on a request's new tokens
  int longest;         // bound on a request's tokens
  // How the tensor-core kernel cuts the rows of a KV head (weigh_plan).
  int few;                        // few rows: K streams through
  int tokens, heads, head_parts;  // a row tile: so many tokens x heads; tiles for the heads of a group
  int cols;                       // its rows, rounded up to the MMA's granularity
  int parts, per_part;            // parts of a request's row tiles, tiles of a part
  int run;                        // jobs that a CTA takes in a row
  float* partial;                 // [parts, hkv, slots], null: one part, added to the weights directly
  // With kv_lo or kv_hi (null: causal) the keys that row tiles and that parts see:
  int4* ranges;     // least and end of any row's, of all rows'
  int2* part_keys;  // [R, parts]
};

constexpr int kWeighFew = 16;    // most rows of a row tile where K streams
constexpr int kWeighRows = 112;  // and of one where many tiles meet the same keys

// Row tiles and parts for these sizes; everything follows from host sizes.
// `slots`: room of all requests.
inline void weigh_plan(WeighArgs& w, int sms) {
  const int G = w.a.G;
  const long long rows = static_cast<long long>(w.most) * G;
  w.few = rows <= kWeighFew;
  const int keys = w.few ? 128 : 256;  // of a job
  w.heads = G < kWeighRows ? G : kWeighRows;
  w.head_parts = (G + w.heads - 1) / w.heads;
  const int fit = kWeighRows / w.heads;
  const int chunks = (w.most + fit - 1) / fit;
  w.tokens = (w.most + chunks - 1) / chunks;  // chunks of even sizes: a short last one costs as much as a full one
  // Where more tokens fill up the MMA's rows they cost nothing.
  int unit = 16;
  while (unit > 1 && unit / 2 * w.heads % 16 == 0) unit /= 2;
  const int full = (w.tokens + unit - 1) / unit * unit;
  if (full <= w.most && full * w.heads <= kWeighRows) w.tokens = full;
  w.cols = (w.tokens * w.heads + 15) / 16 * 16;
  const long long tiles = static_cast<long long>((w.most + w.tokens - 1) / w.tokens) * w.head_parts;
  // Jobs of (keys, part of the rows): enough to even out the SMs, each of at
  // least six row tiles (K is copied once per job).
  const long long key_tiles = (w.slots + keys - 1) / keys, jobs = key_tiles * w.a.L.hkv;
  long long parts = (32ll * sms + jobs - 1) / jobs;
  const long long most = (tiles + 5) / 6;
  parts = parts < most ? parts : most;
  parts = parts < 32 ? parts : 32;
  parts = parts > 1 ? parts : 1;
  w.per_part = static_cast<int>((tiles + parts - 1) / parts);
  w.parts = static_cast<int>((tiles + w.per_part - 1) / w.per_part);
  // Heads of the same keys in a row (the walk is short between them, and their
  // keys lie next to each other), as long as that leaves each CTA many such runs.
  w.run = 1;
  while (w.few && w.a.L.hkv % (2 * w.run) == 0 && jobs >= 32ll * w.run * sms) w.run *= 2;
}

inline size_t weigh_range_bytes(const WeighArgs& w) {
  return ((static_cast<size_t>(w.a.T) / w.tokens + w.a.R + 2) * sizeof(int4) +
          static_cast<size_t>(w.a.R) * w.parts * sizeof(int2) + 15) & ~static_cast<size_t>(15);
}

// Where the token chunks of request r's first token t0 begin in `ranges`.
__host__ __device__ inline long long weigh_range_at(int t0, int r, int tokens) { return t0 / tokens + r; }

int launch_weigh_rows(const WeighArgs& w, int kv_dtype, cudaStream_t stream);
bool weigh_tensor_takes(int kv_dtype, int d, int page_size, const void* k, const void* q, long long q_ts, long long q_hs);
constexpr int kWeighNoMap = -1000;  // (no CUDA error's number) the queries' strides do not fit a tensor map, nothing was launched
int launch_weigh_tensor(const WeighArgs& w, int kv_dtype, int sms, cudaStream_t stream);
int set_wait_limit_weigh(unsigned long long ns);

}  // namespace stk
