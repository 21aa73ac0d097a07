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
  int tokens, heads, head_parts;  // a row tile: so many tokens x heads; tiles for the heads of a group
  int cols;                       // its rows, rounded up to the MMA's granularity
  int parts, per_part;            // parts of a request's row tiles, tiles of a part
  float* partial;                 // [parts, hkv, slots], null: one part, added to the weights directly
  int4* ranges;                   // keys that row tiles see (kv_lo or kv_hi given), null: causal
};

constexpr int kWeighRows = 112;  // most rows of a row tile
constexpr int kWeighKeys = 256;  // keys of a job

// Row tiles and parts for these sizes; everything follows from host sizes.
inline void weigh_plan(WeighArgs& w, long long key_tiles, int sms) {
  const int G = w.a.G;
  w.heads = G < kWeighRows ? G : kWeighRows;
  w.head_parts = (G + w.heads - 1) / w.heads;
  const int fit = kWeighRows / w.heads;
  w.tokens = fit < w.most ? fit : w.most;
  w.cols = (w.tokens * w.heads + 15) / 16 * 16;
  const long long tiles = static_cast<long long>((w.most + w.tokens - 1) / w.tokens) * w.head_parts;
  // Jobs of (256 keys, part of the rows): enough to even out the SMs, each of
  // at least four row tiles.
  const long long jobs = key_tiles * w.a.L.hkv;
  long long parts = (8ll * sms + jobs - 1) / jobs;
  const long long most = (tiles + 3) / 4;
  parts = parts < most ? parts : most;
  parts = parts < 16 ? parts : 16;
  parts = parts > 1 ? parts : 1;
  w.per_part = static_cast<int>((tiles + parts - 1) / parts);
  w.parts = static_cast<int>((tiles + w.per_part - 1) / w.per_part);
}

// Row tiles of token chunks before request r's first, at most.
__host__ __device__ inline long long weigh_range_at(int t0, int r, int tokens) { return t0 / tokens + r; }

int launch_weigh_rows(const WeighArgs& w, int kv_dtype, cudaStream_t stream);
bool weigh_tensor_takes(int kv_dtype, int d, int page_size, const void* k, const void* q, long long q_ts, long long q_hs);
// 1: the queries' strides do not fit a tensor map, nothing was launched.
int launch_weigh_tensor(const WeighArgs& w, int kv_dtype, int sms, cudaStream_t stream);
int set_wait_limit_weigh(unsigned long long ns);

}  // namespace stk
