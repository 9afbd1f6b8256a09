// Attention of drafted tokens: what its kernels are given, and how a request's keys are numbered.
//
// A request of a step holds `held` positions and brings `count` tokens (its nodes), stored behind them in the order they are brought; node i
// stands at positions[i], and of the nodes it sees those that its row of bits names. Of what is held it sees all, or what a window (its own
// position and the window - 1 ahead of it; beside it the first `keep` positions) or a run (its own of `run` positions) leaves.
#pragma once

#include "common.cuh"

struct TreeAttention {
  const void *q, *k_pages, *v_pages, *gate;  // [tokens, nq, d]; key row: k_pages + page * page_stride + (kvh * page_size + off) * d; gate or null
  void* out;                                 // [tokens, nq * dv]
  const int *block_table, *cu_seqlens, *seq_lens, *positions, *ancestors;
  const float* sink;                         // [nq] or null
  float *part_o, *part_ml;                   // [parts, tokens, nq, dv] unnormalised, [parts, tokens, nq, 2] (offset in log2 units, sum)
  int* err;
  long long page_stride;
  int tokens, requests, max_pages, num_pages, nq, nkv, d, dv, page_size, gate_stride, words, window, keep, run, chunk, parts;
  float scale, softcap;
};

// The keys of a request that a step's rows can see, numbered 0, 1, ...: the kept first positions below `lo`, then the positions from `lo` on and
// the nodes behind them. `lo` is where the window or the run of the earliest node, at position `held`, begins.
struct TreeKeys {
  int first, count, held, lo, kept, total;  // first: row of the request's node 0; total: keys, as numbered
  __device__ __forceinline__ int key(int x) const { return x < kept ? x : lo + (x - kept); }
};

__device__ __forceinline__ TreeKeys tree_keys(const TreeAttention& a, int request) {
  TreeKeys k;
  k.first = a.cu_seqlens[request];
  k.count = a.cu_seqlens[request + 1] - k.first;
  const int held = a.seq_lens[request];
  k.held = held - k.count;
  k.lo = k.kept = k.total = 0;
  if (held <= 0 || k.count <= 0) {  // a request that is there for the step's shape only
    k.held = 0;
    return k;
  }
  if (k.held < 0 || k.count > 32 * a.words || k.first < 0 || k.first + k.count > a.tokens) {
    atomicOr(a.err, OMNIA_ERR_WORK);
    k.count = k.first < 0 ? 0 : min(k.count, a.tokens - k.first);
    k.held = 0;
    return k;
  }
  if (a.window > 0) k.lo = max(0, k.held - a.window + 1);
  if (a.run > 0) k.lo = max(k.lo, k.held - k.held % a.run);
  k.kept = min(a.window > 0 ? a.keep : 0, k.lo);
  k.total = k.kept + held - k.lo;
  return k;
}

// The first position that a node at `pos` sees of what is held (beside kept ones).
__device__ __forceinline__ int tree_low(const TreeAttention& a, int pos) {
  int low = a.window > 0 ? pos - a.window + 1 : 0;
  if (a.run > 0) low = max(low, pos - pos % a.run);
  return low;
}
