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

// Equal shares of a step's work for the kernels that keep a fixed number of blocks busy. An item is a tile of rows of one request and one key/value
// head; its keys come in tiles. All tiles of all items stand in one line (requests, then heads, then tiles of rows, then of keys), of which block
// b takes [b T / G, (b + 1) T / G): contexts of unequal lengths cost no block more than another, and since lengths are read here, a captured
// step has its shares right at every replay. An item that several blocks have part in is put together by the merge: block b leaves
// what its first item came to in slot 2 b, and what its last one did in slot 2 b + 1.
constexpr int TREE_MOST_REQUESTS = 1024;

struct TreeShares {
  int rows, keys;  // of a tile
  __device__ __forceinline__ int row_tiles(const TreeAttention& a, const TreeKeys& k) const {
    return k.total > 0 ? (k.count * (a.nq / a.nkv) + rows - 1) / rows : 0;
  }
  __device__ __forceinline__ int key_tiles(const TreeKeys& k) const { return (k.total + keys - 1) / keys; }

  // ends[r]: tiles of all requests up to r, r among them (shared memory, of the whole block); -> tiles in all. `sums`: a word a warp.
  __device__ __forceinline__ long long lay_out(const TreeAttention& a, long long* ends, long long* sums) const {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    long long before = 0;
    for (int r0 = 0; r0 < a.requests; r0 += blockDim.x) {
      const int r = r0 + threadIdx.x;
      long long mine = 0;
      if (r < a.requests) {
        const TreeKeys k = tree_keys(a, r);
        mine = (long long)row_tiles(a, k) * key_tiles(k) * a.nkv;
      }
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const long long other = __shfl_up_sync(0xffffffffu, mine, o);
        if (lane >= o) mine += other;
      }
      if (lane == 31) sums[warp] = mine;
      __syncthreads();
      long long ahead = before;
      for (int w = 0; w < warps; ++w) {
        if (w < warp) ahead += sums[w];
        before += sums[w];
      }
      if (r < a.requests) ends[r] = ahead + mine;
      __syncthreads();
    }
    return before;
  }
};

// A place in that line.
struct TreePlace {
  int request, head, row_tile, tile, row_tiles, tiles;
  TreeKeys k;
  __device__ __forceinline__ void enter(const TreeAttention& a, const TreeShares& s, int r) {
    request = r;
    k = tree_keys(a, r);
    row_tiles = s.row_tiles(a, k), tiles = s.key_tiles(k);
  }
  __device__ __forceinline__ void find(const TreeAttention& a, const TreeShares& s, const long long* ends, long long at) {
    int lo = 0, hi = a.requests - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (ends[mid] > at) hi = mid; else lo = mid + 1;
    }
    enter(a, s, lo);
    const long long in = at - (lo ? ends[lo - 1] : 0);
    const int each = row_tiles * tiles;
    head = (int)(in / each);
    const int rest = (int)(in % each);
    row_tile = rest / tiles, tile = rest % tiles;
  }
  // To the next tile, which there is.
  __device__ __forceinline__ void next(const TreeAttention& a, const TreeShares& s) {
    if (++tile < tiles) return;
    tile = 0;
    if (++row_tile < row_tiles) return;
    row_tile = 0;
    if (++head < a.nkv) return;
    head = 0;
    do enter(a, s, request + 1);
    while (row_tiles * tiles == 0 && request + 1 < a.requests);
  }
};
