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
  int4* items;                               // [requests, nkv, parts], of the kernels by equal shares: where the join finds an item (tree_note)
  long long page_stride;
  // chunk, parts: of the kernel for any shape; by equal shares `parts` is the most tiles of rows that a request has.
  int tokens, requests, max_pages, num_pages, nq, nkv, d, dv, page_size, gate_stride, words, window, keep, run, chunk, parts;
  float scale, softcap;
};

// The keys of a request that a step's rows can see, numbered 0, 1, ...: the kept first positions below `lo`, then the positions from `lo` on and
// the nodes behind them. `lo` is where the window or the run of the earliest node, at position `held`, begins. For a kernel that fetches keys
// `align` at a time, from a multiple of that on, both are rounded to such multiples (what that lets in no row sees).
struct TreeKeys {
  int first, count, held, lo, kept, total;  // first: row of the request's node 0; total: keys, as numbered
  __device__ __forceinline__ int key(int x) const { return x < kept ? x : lo + (x - kept); }
};

__device__ __forceinline__ TreeKeys tree_keys(const TreeAttention& a, int request, int align = 1) {
  TreeKeys k;
  k.first = a.cu_seqlens[request];
  k.count = a.cu_seqlens[request + 1] - k.first;
  const int held = a.seq_lens[request];
  k.held = held - k.count;
  k.lo = k.kept = k.total = 0;
  // Rows that are not the step's (also of a request that sees nothing, whose zeros are written), or more than there are bits for.
  if (k.first < 0 || k.count < 0 || k.count > a.tokens - k.first || (held > 0 && (k.held < 0 || k.count > 32 * a.words))) {
    atomicOr(a.err, OMNIA_ERR_WORK);
    k.count = k.first < 0 ? 0 : max(0, min(k.count, a.tokens - k.first));
    k.held = 0;
    return k;
  }
  if (held <= 0 || k.count == 0) {  // a request that is there for the step's shape only
    k.held = 0;
    return k;
  }
  if (a.window > 0) k.lo = max(0, k.held - a.window + 1);
  if (a.run > 0) k.lo = max(k.lo, k.held - k.held % a.run);
  k.lo -= k.lo % align;
  k.kept = min(a.window > 0 ? (a.keep + align - 1) / align * align : 0, k.lo);
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
// head; its keys come in tiles. All tiles of all items stand in one line (requests, then heads, then tiles of rows, then of keys), ahead of each
// item's as many empty places as its beginning and end cost in tiles, and block b takes [b T / G, (b + 1) T / G) of the T places: contexts of unequal lengths
// cost no block more than another, and since lengths are read here, a captured step has its shares right at every replay. An item that several
// blocks have part in is put together by the join: block b leaves in slot 2 b what the item came to that the block begins in (or ahead of, in its empty
// places), and in slot 2 b + 1 what its last one did.
constexpr int TREE_MOST_REQUESTS = 1024;

struct TreeShares {
  int rows, keys, align, extra;  // rows and keys of a tile; of `tree_keys`; empty places ahead of an item
  __device__ __forceinline__ int row_tiles(const TreeAttention& a, const TreeKeys& k) const {
    return k.total > 0 ? (k.count * (a.nq / a.nkv) + rows - 1) / rows : 0;
  }
  __device__ __forceinline__ int key_tiles(const TreeKeys& k) const { return (k.total + keys - 1) / keys; }

  __device__ __forceinline__ long long places(const TreeAttention& a, const TreeKeys& k) const {
    return k.total > 0 ? (long long)row_tiles(a, k) * (key_tiles(k) + extra) * a.nkv : 0;
  }

  // ends[r]: places of all requests up to r, r among them (shared memory, of the whole block); -> places in all. `sums`: a word a warp.
  __device__ __forceinline__ long long lay_out(const TreeAttention& a, long long* ends, long long* sums) const {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    long long before = 0;
    for (int r0 = 0; r0 < a.requests; r0 += blockDim.x) {
      const int r = r0 + threadIdx.x;
      long long mine = 0;
      if (r < a.requests) {
        mine = places(a, tree_keys(a, r, align));
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

// A tile in that line, and how many places from it on are the block's (0: there is none).
struct TreePlace {
  int request, head, row_tile, tile, row_tiles, tiles, left;
  TreeKeys k;
  __device__ __forceinline__ void enter(const TreeAttention& a, const TreeShares& s, int r) {
    request = r;
    k = tree_keys(a, r, s.align);
    row_tiles = s.row_tiles(a, k), tiles = s.key_tiles(k);
  }
  // The first tile of the `share` places from `at` on. -> where its item's places begin
  __device__ __forceinline__ long long find(const TreeAttention& a, const TreeShares& s, const long long* ends, long long at, int share) {
    int lo = 0, hi = a.requests - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (ends[mid] > at) hi = mid; else lo = mid + 1;
    }
    enter(a, s, lo);
    const long long in = at - (lo ? ends[lo - 1] : 0);
    const int item = tiles + s.extra, each = row_tiles * item;
    head = (int)(in / each);
    const int rest = (int)(in % each);
    row_tile = rest / item, tile = rest % item - s.extra;
    const long long begin = at - (tile + s.extra);
    left = share;
    if (tile < 0) left = max(left + tile, 0), tile = 0;
    return begin;
  }
  // `count` tiles on, to the next item at most.
  __device__ __forceinline__ void next(const TreeAttention& a, const TreeShares& s, int count = 1) {
    left -= count, tile += count;
    if (tile < tiles) return;
    left = max(left - s.extra, 0), tile = 0;
    if (left == 0) return;
    if (++row_tile < row_tiles) return;
    row_tile = 0;
    if (++head < a.nkv) return;
    head = 0;
    do enter(a, s, request + 1);
    while (row_tiles * tiles == 0 && request + 1 < a.requests);
  }
};

// Where the join finds an item, by the block that has its first tile and whose share of the line ends at place `upto` (one thread of it): in how many
// pieces it is, in which slot the first one is, in which the next (one a block from there on).
__device__ __forceinline__ void tree_note(const TreeAttention& a, long long total, long long blocks, long long upto, const TreePlace& now, bool first) {
  if (now.row_tile >= a.parts) return;  // (more nodes than the call allows for, which the join reports)
  const int block = blockIdx.x;
  int4 item = make_int4(1, 0, 0, 0);
  if (now.tiles > now.left) {
    const long long last = ((upto - now.left + now.tiles) * blocks - 1) / total;  // the block that has the item's last tile
    item = make_int4((int)last - block + 1, 2 * block + (first ? 0 : 1), 2 * block + 2, 0);
  }
  a.items[((size_t)now.request * a.nkv + now.head) * a.parts + now.row_tile] = item;
}

constexpr int TREE_JOIN_WARPS = 4;

__device__ __forceinline__ float tree_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// sigmoid(x) to some units of float32's last place.
__device__ __forceinline__ float tree_sigmoid(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(1.f + tree_exp2(-1.4426950408889634f * x)));
  return y;
}
__device__ __forceinline__ unsigned tree_pair(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const unsigned*>(&v);
}

// An item that several blocks had part in, put together: a warp a row, the slots in the order of their blocks, eight on their way at once, the sink, the
// gate. Bytes: 4 (D + 2) a row and piece, out of L2; what it takes, 3 to 5 us behind the kernel ahead, is the wait, where the item lies, and a round trip
// for eight pieces. (Blocks by the borders of the kernel's blocks, most of which had nothing to do: 10 us for 592 blocks of 12 items' rows.) Offsets, sums and
// what is summed are float32; one rounding to the output's type. A block of the grid's first axis has an item (a request's first one: its zeros, where it sees nothing), whose rows the second axis shares out. What
// is read ahead of the wait was there ahead of the kernel that this one waits for. `slots`: how many there are.
template <typename T, int MOST>
__global__ void __launch_bounds__(32 * TREE_JOIN_WARPS) tree_join_kernel(const __grid_constant__ TreeAttention a, const TreeShares shares, int slots, int most) {
  constexpr int WARPS = TREE_JOIN_WARPS, PER = (MOST + 127) / 128;  // four dims a lane
  constexpr float LOG2E = 1.4426950408889634f;
  const int D = a.d;  // a multiple of 4, MOST at most
  const int group = a.nq / a.nkv, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, step = WARPS * gridDim.y, r0 = blockIdx.y * WARPS + warp;
  const int request = blockIdx.x / (a.nkv * a.parts), within = blockIdx.x % (a.nkv * a.parts), kvh = within / a.parts, row0 = within % a.parts * shares.rows;
  const TreeKeys k = tree_keys(a, request, shares.align);
  if (k.count > most && within == 0 && blockIdx.y == 0 && threadIdx.x == 0) atomicOr(a.err, OMNIA_ERR_WORK);
  const int rows = k.total > 0 ? min(shares.rows, k.count * group - row0) : 0;
  float gates[PER][4], sink = 0.f;
  auto ahead = [&](int r) {  // what a row needs beside its pieces
    if (r >= rows) return;
    const int in = row0 + r, token = k.first + in / group, head = kvh * group + in % group;
    sink = a.sink ? a.sink[head] * LOG2E : -INFINITY;
#pragma unroll
    for (int i = 0; i < PER; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = (32 * i + lane) * 4 + j;
        gates[i][j] = a.gate && c < D ? to_f32(static_cast<const T*>(a.gate)[(size_t)token * a.gate_stride + head * D + c]) : 0.f;
      }
  };
  ahead(r0);
  pdl_wait();
  pdl_launch_dependents();
  if (k.total <= 0) {
    if (within > 0) return;
    for (int r = r0; r < k.count * a.nq; r += step)
      for (int c = lane; c < D; c += 32) static_cast<T*>(a.out)[((size_t)k.first * a.nq + r) * D + c] = from_f32<T>(0.f);
    return;
  }
  if (rows <= 0) return;
  const int4 item = a.items[blockIdx.x];
  const int parts = item.x;
  // One piece is its block's to write. (What lies outside the slots a kernel that gave up has left unwritten.)
  if (parts < 2 || parts > slots || item.y < 0 || item.y >= slots || item.z < 0 || item.z + 2 * (parts - 2) >= slots) return;
  for (int r = r0; r < rows; r += step) {
    const int in = row0 + r, token = k.first + in / group, head = kvh * group + in % group;
    if (r > r0) ahead(r);
    float4 sum[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) sum[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    float base = -INFINITY, l = 0.f;
    for (int p0 = 0; p0 < parts; p0 += 8) {
      float2 ml[8];
      float4 x[8][PER];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int p = p0 + u;
        const size_t row = (size_t)(p == 0 ? item.y : item.z + 2 * (p - 1)) * shares.rows + r;
        ml[u] = p < parts ? reinterpret_cast<const float2*>(a.part_ml)[row] : make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int c = (32 * i + lane) * 4;
          x[u][i] = p < parts && c < D ? *reinterpret_cast<const float4*>(a.part_o + row * D + c) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
      }
      float over = base;
#pragma unroll
      for (int u = 0; u < 8; ++u) over = fmaxf(over, ml[u].x);
      const float offset = over == -INFINITY ? 0.f : over, f = tree_exp2(base - offset);
      base = over, l *= f;
#pragma unroll
      for (int i = 0; i < PER; ++i) sum[i].x *= f, sum[i].y *= f, sum[i].z *= f, sum[i].w *= f;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float w = tree_exp2(ml[u].x - offset);
        l = fmaf(ml[u].y, w, l);  // (no number where a row's scores are none: their maximum is then -infinity)
        if (w == 0.f) continue;   // (what it came to then need not be a number)
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          sum[i].x = fmaf(x[u][i].x, w, sum[i].x), sum[i].y = fmaf(x[u][i].y, w, sum[i].y);
          sum[i].z = fmaf(x[u][i].z, w, sum[i].z), sum[i].w = fmaf(x[u][i].w, w, sum[i].w);
        }
      }
    }
    const float over = fmaxf(base, sink), offset = over == -INFINITY ? 0.f : over, f = tree_exp2(base - offset);
    l = l * f + tree_exp2(sink - offset);
    const float by = l > 0.f || l != l ? f / l : 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = (32 * i + lane) * 4;
      if (c >= D) continue;
      float y[4] = {sum[i].x * by, sum[i].y * by, sum[i].z * by, sum[i].w * by};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (by == 0.f) y[j] = 0.f;
        if (a.gate) y[j] *= tree_sigmoid(gates[i][j]);
      }
      T* to = static_cast<T*>(a.out) + (size_t)token * a.nq * D + head * D + c;
      if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(to) = make_uint2(tree_pair(y[0], y[1]), tree_pair(y[2], y[3]));
      else *reinterpret_cast<float4*>(to) = make_float4(y[0], y[1], y[2], y[3]);
    }
  }
  OMNIA_TRACE_BLOCK(7);  // the rows are out
}

// The most tiles of rows that a request has.
inline int tree_row_tiles(const TreeAttention& a, int most_nodes, int rows) { return (most_nodes * (a.nq / a.nkv) + rows - 1) / rows; }

// (`a.parts` is that number.)
template <typename T, int MOST>
int tree_join(const TreeAttention& a, const TreeShares& shares, int most_nodes, int blocks, cudaStream_t stream) {
  const int rows = min(shares.rows, most_nodes * (a.nq / a.nkv)), items = a.requests * a.nkv * a.parts;
  // A warp a row as long as blocks that have little to do are not many times what the GPU holds at once.
  const dim3 grid(items, max(1, min(min((rows + TREE_JOIN_WARPS - 1) / TREE_JOIN_WARPS, 16), 4096 / items)));
  launch_pdl(tree_join_kernel<T, MOST>, grid, dim3(32 * TREE_JOIN_WARPS), 0, stream, a, shares, 2 * blocks, most_nodes);
  return OMNIA_LAUNCH_RESULT();
}
