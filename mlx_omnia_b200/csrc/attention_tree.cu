// Attention of trees of drafted tokens for any head sizes (<= 512; keys and values may differ in width), page size, element type and number of requests, with
// the merge of its pieces, and the 32-bit path's kernel by equal shares (whose items the join of attention_tree.cuh puts together).
//
//   out[i, h] = sigmoid(gate) * sum_k p_k v_k / (sum_k p_k + exp(sink_h)),  p_k = exp(s_k), s_k = scale q_i . k (softcap tanh(s / softcap))
//
// over the keys that node i sees (attention_tree.cuh); a node that sees nothing has zeros.
//
// The rows of a tile are (node, query head of the group) pairs of one key/value head, so that a key fetched is used by all of them. A block
// has a tile of 32 rows and a run of `chunk` keys, which it walks in tiles held in shared memory as float32, with the softmax's
// maximum and sum kept along; products run on the ordinary float32 units, a thread 4 rows x 4 keys and 4 rows x D / 16 dims. It is here for
// the sizes that no other kernel takes (widths of keys and values that differ, that are no multiple of 4 or 8, heads above 256); all that it holds is float32. With more than one
// chunk a block writes its maximum, sum and unnormalised sums to memory and the merge adds them in the chunks' order, so the
// result does not depend on which block was first.
//
// The 32-bit path's kernel (keys and values of one width, a multiple of 4 up to 256) does the same products, but works off equal shares of the step's tiles
// (TreeShares), its tiles coming by cp.async while the one before is at work. What bounds long steps is the float32 units and the shared memory that feeds them, a 16-byte read for 4 to 8 operations: 16 requests of
// 3,000 positions with 32 tokens, 4 heads of 128: 498 us, 25 TFLOP/s. Short ones end at a tile's chain of reads: 12 requests of 1,001 with 13 tokens, 8 query
// heads of 24 to one, 20.3 us, of them 11 to the last tile's sums (shares known after 2.7, the tile there after 6.4, its scores at 9).
#include "attention_tree.cuh"

namespace {

constexpr int THREADS = 128, ROWS = 32;
constexpr float LOG2E = 1.4426950408889634f;

// Of the kernel for any shape: one thread a request and key/value head.
__device__ __forceinline__ bool tid0() { return threadIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0; }

template <typename T>
__device__ __forceinline__ void finish_dim(const TreeAttention& a, int token, int head, int dim, float value) {
  if (a.gate) {
    const float g = to_f32(static_cast<const T*>(a.gate)[(size_t)token * a.gate_stride + head * a.dv + dim]);
    value *= 1.f / (1.f + expf(-g));
  }
  static_cast<T*>(a.out)[(size_t)token * a.nq * a.dv + head * a.dv + dim] = from_f32<T>(value);
}

// MOST: a multiple of 64 that neither width exceeds; KEYS: keys of a tile.
template <typename T, int MOST, int KEYS>
__global__ void __launch_bounds__(THREADS) tree_pieces_kernel(const __grid_constant__ TreeAttention a) {
  constexpr int STRIDE = MOST + 4, DIMS = MOST / 16, PER = KEYS / 16;  // floats of a row in shared memory; dims, keys of a thread
  extern __shared__ __align__(16) float smem[];
  float *qs = smem, *ks = qs + ROWS * STRIDE, *vs = ks + KEYS * STRIDE, *ps = vs + KEYS * STRIDE;  // ps [KEYS][ROWS + 4]
  __shared__ int low[ROWS], node_pos[KEYS], key_of[KEYS], off_of[KEYS];
  __shared__ long long page_of[KEYS];  // elements from the pages' beginning
  __shared__ float top[ROWS], sum[ROWS], factor[ROWS];
  pdl_wait();
  pdl_launch_dependents();
  const int request = blockIdx.x / a.nkv, kvh = blockIdx.x % a.nkv, part = blockIdx.z, group = a.nq / a.nkv;
  const TreeKeys k = tree_keys(a, request);
  if ((k.total > (long long)a.parts * a.chunk || k.count * group > (int)gridDim.y * ROWS) && tid0()) atomicOr(a.err, OMNIA_ERR_WORK);
  const int rows = k.count * group, row0 = blockIdx.y * ROWS, here = min(rows - row0, ROWS);
  if (here <= 0) return;
  const int x0 = part * a.chunk, x1 = min(x0 + a.chunk, k.total);
  if (x0 >= x1 && part > 0) return;
  const int tid = threadIdx.x;
  const T *q = static_cast<const T*>(a.q), *kp = static_cast<const T*>(a.k_pages), *vp = static_cast<const T*>(a.v_pages);
  for (int i = tid; i < ROWS * MOST; i += THREADS) {
    const int r = i / MOST, c = i % MOST, row = row0 + r;
    float v = 0.f;
    if (r < here && c < a.d) v = to_f32(q[((size_t)(k.first + row / group) * a.nq + kvh * group + row % group) * a.d + c]) * a.scale;
    qs[r * STRIDE + c] = v;
  }
  if (tid < ROWS) {
    top[tid] = -INFINITY, sum[tid] = 0.f;
    low[tid] = tid < here ? tree_low(a, a.positions[k.first + (row0 + tid) / group]) : 0;
  }
  const int rg = tid / 16, cg = tid % 16;  // this thread's rows 4 rg .. 4 rg + 3; its keys or dims: cg, cg + 16, ...
  float acc[4][DIMS];
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int c = 0; c < DIMS; ++c) acc[r][c] = 0.f;
  const int* table = a.block_table + (size_t)request * a.max_pages;
  const bool pieces = a.d * sizeof(T) % 16 == 0 && a.dv * sizeof(T) % 16 == 0 && a.page_stride * sizeof(T) % 16 == 0 &&
                      ((reinterpret_cast<uintptr_t>(kp) | reinterpret_cast<uintptr_t>(vp)) & 15) == 0;
  // Columns beyond the widths: no load writes them.
  for (int i = tid; i < KEYS * (MOST - max(a.d, a.dv)); i += THREADS) {
    const int t = i / (MOST - max(a.d, a.dv)), c = max(a.d, a.dv) + i % (MOST - max(a.d, a.dv));
    ks[t * STRIDE + c] = vs[t * STRIDE + c] = 0.f;
  }
  for (int x = x0; x < x1; x += KEYS) {
    __syncthreads();
    if (tid < KEYS) {
      int key = -1, pos = 0;
      if (x + tid < x1) {
        key = k.key(x + tid);
        const int page = key / a.page_size;
        pos = key < k.held ? key : a.positions[k.first + key - k.held];
        const int at = page < a.max_pages ? table[page] : -1;
        if (at < 0 || at >= a.num_pages) atomicOr(a.err, OMNIA_ERR_PAGE), key = -1;
        page_of[tid] = at * a.page_stride, off_of[tid] = kvh * a.page_size + key % a.page_size;
      }
      key_of[tid] = key, node_pos[tid] = pos;
    }
    __syncthreads();
    bool odd = false;  // whether a value is no finite number: what a row does not see then stays out of its sums by a test, for 0 x NaN is NaN
    // Rows in pieces of 16 bytes where they are made of such, four pieces of keys and of values on their way at once.
    constexpr int PIECE = 16 / sizeof(T);
    if (pieces) {
      const int wide = max(a.d, a.dv) / PIECE;
      for (int i0 = tid; i0 < KEYS * wide; i0 += 4 * THREADS) {
        uint4 k4[4], v4[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int i = i0 + u * THREADS, t = i / wide, c = (i - t * wide) * PIECE;
          k4[u] = v4[u] = make_uint4(0u, 0u, 0u, 0u);
          if (i < KEYS * wide && key_of[t] >= 0) {
            if (c < a.d) k4[u] = *reinterpret_cast<const uint4*>(kp + page_of[t] + (long long)off_of[t] * a.d + c);
            if (c < a.dv) v4[u] = *reinterpret_cast<const uint4*>(vp + page_of[t] + (long long)off_of[t] * a.dv + c);
          }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int i = i0 + u * THREADS, t = i / wide, c = (i - t * wide) * PIECE;
          if (i >= KEYS * wide) continue;
          const T *kx = reinterpret_cast<const T*>(&k4[u]), *vx = reinterpret_cast<const T*>(&v4[u]);
#pragma unroll
          for (int e = 0; e < PIECE; ++e) {
            const float v = to_f32(vx[e]);
            ks[t * STRIDE + c + e] = to_f32(kx[e]), vs[t * STRIDE + c + e] = v;
            odd |= !(fabsf(v) < INFINITY);
          }
        }
      }
    } else {
      const int wide = max(a.d, a.dv);
#pragma unroll 4
      for (int i = tid; i < KEYS * wide; i += THREADS) {
        const int t = i / wide, c = i - t * wide;
        const bool there = key_of[t] >= 0;
        const float v = there && c < a.dv ? to_f32(vp[page_of[t] + (long long)off_of[t] * a.dv + c]) : 0.f;
        ks[t * STRIDE + c] = there && c < a.d ? to_f32(kp[page_of[t] + (long long)off_of[t] * a.d + c]) : 0.f;
        vs[t * STRIDE + c] = v;
        odd |= !(fabsf(v) < INFINITY);
      }
    }
    const bool careful = __syncthreads_or(odd);
    float s[4][PER];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int t = 0; t < PER; ++t) s[r][t] = 0.f;
    for (int c = 0; c < a.d; c += 4) {
      float4 kf[PER], qf[4];
#pragma unroll
      for (int t = 0; t < PER; ++t) kf[t] = *reinterpret_cast<const float4*>(ks + (cg + 16 * t) * STRIDE + c);
#pragma unroll
      for (int r = 0; r < 4; ++r) qf[r] = *reinterpret_cast<const float4*>(qs + (4 * rg + r) * STRIDE + c);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int t = 0; t < PER; ++t)
          s[r][t] = fmaf(qf[r].w, kf[t].w, fmaf(qf[r].z, kf[t].z, fmaf(qf[r].y, kf[t].y, fmaf(qf[r].x, kf[t].x, s[r][t]))));
    }
    // What a row does not see has no weight. A row's scores lie with sixteen neighbouring lanes.
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int mine = 4 * rg + r, node = (row0 + mine) / group;
      const int least = low[mine];
      float most = -INFINITY;
#pragma unroll
      for (int t = 0; t < PER; ++t) {
        const int at = cg + 16 * t, key = key_of[at], pos = node_pos[at];
        bool seen = mine < here && key >= 0 && (pos >= least || (a.window > 0 && pos < a.keep));
        if (seen && key >= k.held) {
          const int m = key - k.held;
          seen = ((unsigned)a.ancestors[(size_t)(k.first + node) * a.words + (m >> 5)] >> (m & 31)) & 1u;
        }
        if (a.softcap > 0.f) s[r][t] = a.softcap * tanhf(s[r][t] / a.softcap);
        s[r][t] = seen ? s[r][t] * LOG2E : -INFINITY;
        most = fmaxf(most, s[r][t]);
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
      const float old = top[mine], now = fmaxf(old, most), base = now == -INFINITY ? 0.f : now;
      float total = 0.f;
#pragma unroll
      for (int t = 0; t < PER; ++t) {
        const float p = exp2f(s[r][t] - base);
        total += p;
        ps[(cg + 16 * t) * (ROWS + 4) + mine] = p;
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
      __syncwarp();
      if (cg == 0) {
        const float f = exp2f(old - base);
        factor[mine] = f, sum[mine] = sum[mine] * f + total, top[mine] = now;
      }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float f = factor[4 * rg + r];
#pragma unroll
      for (int c = 0; c < DIMS; ++c) acc[r][c] *= f;
    }
    if (careful) {
      for (int t = 0; t < KEYS; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float p = ps[t * (ROWS + 4) + 4 * rg + r];
          if (p == 0.f) continue;
#pragma unroll
          for (int c = 0; c < DIMS; ++c) acc[r][c] = fmaf(p, vs[t * STRIDE + cg + 16 * c], acc[r][c]);
        }
      continue;
    }
    for (int t = 0; t < KEYS; ++t) {
      const float4 p = *reinterpret_cast<const float4*>(ps + t * (ROWS + 4) + 4 * rg);
#pragma unroll
      for (int c = 0; c < DIMS; ++c) {
        const float v = vs[t * STRIDE + cg + 16 * c];
        acc[0][c] = fmaf(p.x, v, acc[0][c]), acc[1][c] = fmaf(p.y, v, acc[1][c]);
        acc[2][c] = fmaf(p.z, v, acc[2][c]), acc[3][c] = fmaf(p.w, v, acc[3][c]);
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int mine = 4 * rg + r, row = row0 + mine;
    if (mine >= here) continue;
    const int token = k.first + row / group, head = kvh * group + row % group;
    if (a.parts > 1) {
      const size_t at = ((size_t)part * a.tokens + token) * a.nq + head;
      if (cg == 0) a.part_ml[2 * at] = top[mine], a.part_ml[2 * at + 1] = sum[mine];
#pragma unroll
      for (int c = 0; c < DIMS; ++c)
        if (cg + 16 * c < a.dv) a.part_o[at * a.dv + cg + 16 * c] = acc[r][c];
      continue;
    }
    float l = sum[mine], f = 1.f;
    if (a.sink) {
      const float z = a.sink[head] * LOG2E, base = fmaxf(top[mine], z);
      f = exp2f(top[mine] - base), l = l * f + exp2f(z - base);
    }
    const float unit = l > 0.f || l != l ? f / l : 0.f;
#pragma unroll
    for (int c = 0; c < DIMS; ++c)
      if (cg + 16 * c < a.dv) finish_dim<T>(a, token, head, cg + 16 * c, acc[r][c] * unit);
  }
}

// The 32-bit path. MOST: a multiple of 32 that the width does not exceed.
template <int MOST>
struct Shares32 {
  static constexpr int KEYS = MOST <= 64 ? 64 : 32, STRIDE = MOST + 4, PER = KEYS / 16, DIMS = MOST / 16, EXTRA = 2;
  static constexpr int PLACES = MOST <= 32 ? 4 : MOST <= 128 ? 2 : 1;  // blocks of an SM
  static constexpr int FLOATS = ROWS * STRIDE + 4 * KEYS * STRIDE + KEYS * (ROWS + 4);
  static_assert(FLOATS * sizeof(float) >= TREE_MOST_REQUESTS * sizeof(long long), "the requests' ends lie where the tiles are to be");
};
template <int MOST>
__global__ void __launch_bounds__(THREADS, Shares32<MOST>::PLACES) tree_shares32_kernel(const __grid_constant__ TreeAttention a) {
  using S = Shares32<MOST>;
  constexpr int KEYS = S::KEYS, STRIDE = S::STRIDE, PER = S::PER, DIMS = S::DIMS, WARPS = THREADS / 32, MINE = KEYS / WARPS;
  extern __shared__ __align__(16) float smem[];
  float *qs = smem, *stages = qs + ROWS * STRIDE, *ps = stages + 4 * KEYS * STRIDE;  // stages: keys, values, of two tiles; ps [KEYS][ROWS + 4]
  long long* ends = reinterpret_cast<long long*>(smem);
  __shared__ long long sums[WARPS];
  __shared__ int low[ROWS];
  __shared__ float top[ROWS], sum[ROWS];
  pdl_wait();
  pdl_launch_dependents();
  const TreeShares shares = {ROWS, KEYS, 1, S::EXTRA};
  const long long total = shares.lay_out(a, ends, sums), blocks = min((long long)gridDim.x, total);
  if (blockIdx.x >= blocks) return;
  const long long t0 = total * blockIdx.x / blocks, upto = total * (blockIdx.x + 1) / blocks;
  TreePlace ahead;
  ahead.find(a, shares, ends, t0, (int)(upto - t0));
  if (ahead.left == 0) return;
  TreePlace now = ahead;
  __syncthreads();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, group = a.nq / a.nkv, d = a.d;
  for (int i = tid; i < (ROWS + 4 * KEYS) * (MOST - d); i += THREADS)  // the columns beyond a row: no load writes them
    smem[i / (MOST - d) * STRIDE + d + i % (MOST - d)] = 0.f;
  const float *q = static_cast<const float*>(a.q), *kp = static_cast<const float*>(a.k_pages);
  const long long apart = static_cast<const float*>(a.v_pages) - kp;

  // Lane l < MINE knows where the l-th row of its warp's share of the tile at `ahead` lies.
  auto where = [&]() -> long long {
    const int x = ahead.tile * KEYS + warp * MINE + lane;
    if (lane >= MINE || x >= ahead.k.total) return -1;
    const int key = ahead.k.key(x), at = key / a.page_size;
    const int page = at < a.max_pages ? a.block_table[(size_t)ahead.request * a.max_pages + at] : -1;
    if (page < 0 || page >= a.num_pages) {
      atomicOr(a.err, OMNIA_ERR_PAGE);
      return -1;
    }
    return page * a.page_stride + (long long)(ahead.head * a.page_size + key % a.page_size) * d;
  };
  long long row_at = where();
  int load_stage = 0;
  auto fetch = [&]() {  // the tile at `ahead`, into the next stage; then on
    if (ahead.left > 0) {
      float* k_s = stages + load_stage * 2 * KEYS * STRIDE + warp * MINE * STRIDE;
      load_stage ^= 1;
      constexpr int ACROSS = MOST / 4, PIECES = MINE * ACROSS;
#pragma unroll 4
      for (int i0 = 0; i0 < PIECES; i0 += 32) {
        const int i = i0 + lane, row = i / ACROSS, c = i % ACROSS * 4;
        const long long from = __shfl_sync(0xffffffffu, row_at, row);
        if (c >= d) continue;
        const unsigned to = (unsigned)__cvta_generic_to_shared(k_s + row * STRIDE + c);
        const float* at = kp + (from < 0 ? 0 : from) + c;
        const int bytes = from < 0 ? 0 : 16;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(to), "l"(at), "r"(bytes) : "memory");
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(to + KEYS * STRIDE * 4), "l"(at + apart), "r"(bytes) : "memory");
      }
      ahead.next(a, shares);
      if (ahead.left > 0) row_at = where();
    }
    asm volatile("cp.async.commit_group;\n" ::: "memory");
  };
  fetch();

  const int rg = tid / 16, cg = tid % 16;  // this thread's rows 4 rg .. 4 rg + 3; its keys: cg, cg + 16, ...; its dims: DIMS from DIMS cg on, or 4 from 4 cg + 64 c on
  constexpr int RUN = DIMS < 4 ? DIMS : 4;
  float acc[4][DIMS];
  const bool halfway = now.tile > 0;
  bool first = true, entered = true;
  int stage = 0;
  while (now.left > 0) {
    const int rows = now.k.count * group, row0 = now.row_tile * ROWS, here = min(ROWS, rows - row0);
    if (entered) {
      if (tid == 0 && now.tile == 0) tree_note(a, total, blocks, upto, now, first);
      for (int i = tid; i < ROWS * (MOST / 4); i += THREADS) {
        const int r = i / (MOST / 4), c = i % (MOST / 4) * 4, row = row0 + r;
        if (c >= d) continue;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if (r < here) {
          const float* from = q + ((size_t)(now.k.first + row / group) * a.nq + now.head * group + row % group) * d + c;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = from[e] * a.scale;
        }
        *reinterpret_cast<float4*>(qs + r * STRIDE + c) = make_float4(v[0], v[1], v[2], v[3]);
      }
      if (tid < ROWS) {
        top[tid] = -INFINITY, sum[tid] = 0.f;
        low[tid] = tid < here ? tree_low(a, a.positions[now.k.first + (row0 + tid) / group]) : 0;
      }
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < DIMS; ++c) acc[r][c] = 0.f;
      entered = false;
    }
    asm volatile("cp.async.wait_group 0;\n" ::: "memory");
    __syncthreads();
    fetch();
    const float *ks = stages + stage * 2 * KEYS * STRIDE, *vs = ks + KEYS * STRIDE;
    stage ^= 1;
    float s[4][PER];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int t = 0; t < PER; ++t) s[r][t] = 0.f;
#pragma unroll 4
    for (int c = 0; c < d; c += 4) {
      float4 kf[PER], qf[4];
#pragma unroll
      for (int t = 0; t < PER; ++t) kf[t] = *reinterpret_cast<const float4*>(ks + (cg + 16 * t) * STRIDE + c);
#pragma unroll
      for (int r = 0; r < 4; ++r) qf[r] = *reinterpret_cast<const float4*>(qs + (4 * rg + r) * STRIDE + c);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int t = 0; t < PER; ++t)
          s[r][t] = fmaf(qf[r].w, kf[t].w, fmaf(qf[r].z, kf[t].z, fmaf(qf[r].y, kf[t].y, fmaf(qf[r].x, kf[t].x, s[r][t]))));
    }
    if (a.softcap > 0.f) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int t = 0; t < PER; ++t) s[r][t] = a.softcap * tanhf(s[r][t] / a.softcap);
    }
    // What a row does not see has no weight (where all rows see all keys of the tile there is nothing to ask).
    const int x0 = now.tile * KEYS, last_key = now.k.key(min(x0 + KEYS, now.k.total) - 1);
    const bool clear = x0 + KEYS <= now.k.total && last_key < now.k.held && x0 >= now.k.kept && now.k.key(x0) >= tree_low(a, now.k.held + now.k.count - 1);
    bool careful = false;
    if (!clear) {
#pragma unroll
      for (int t = 0; t < PER; ++t) {
        const int x = x0 + cg + 16 * t;
        int pos = 0, which = -1;
        const bool real = x < now.k.total;
        if (real) {
          pos = now.k.key(x);
          if (pos >= now.k.held) which = pos - now.k.held, pos = a.positions[now.k.first + which];
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int mine = 4 * rg + r;
          bool seen = real && mine < here && (pos >= low[mine] || (a.window > 0 && pos < a.keep));
          if (seen && which >= 0)
            seen = ((unsigned)a.ancestors[(size_t)(now.k.first + (row0 + mine) / group) * a.words + (which >> 5)] >> (which & 31)) & 1u;
          if (!seen) s[r][t] = -INFINITY;
        }
      }
      bool odd = false;  // whether a value is no finite number: what a row does not see then stays out of its sums by a test, for 0 x NaN is NaN
      for (int i = tid; i < KEYS * MOST; i += THREADS) odd |= !(fabsf(vs[i / MOST * STRIDE + i % MOST]) < INFINITY);
      careful = __syncthreads_or(odd);
    }
    // A row's scores lie with sixteen neighbouring lanes; the four rows go side by side.
    float most[4], old[4], base[4], all[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      most[r] = -INFINITY, old[r] = top[4 * rg + r], all[r] = 0.f;
#pragma unroll
      for (int t = 0; t < PER; ++t) s[r][t] *= LOG2E, most[r] = fmaxf(most[r], s[r][t]);
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1)
#pragma unroll
      for (int r = 0; r < 4; ++r) most[r] = fmaxf(most[r], __shfl_xor_sync(0xffffffffu, most[r], o));
#pragma unroll
    for (int r = 0; r < 4; ++r) most[r] = fmaxf(old[r], most[r]), base[r] = most[r] == -INFINITY ? 0.f : most[r];
#pragma unroll
    for (int t = 0; t < PER; ++t) {
      float p[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) p[r] = exp2f(s[r][t] - base[r]), all[r] += p[r];
      *reinterpret_cast<float4*>(ps + (cg + 16 * t) * (ROWS + 4) + 4 * rg) = make_float4(p[0], p[1], p[2], p[3]);
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1)
#pragma unroll
      for (int r = 0; r < 4; ++r) all[r] += __shfl_xor_sync(0xffffffffu, all[r], o);
    float f[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) f[r] = exp2f(old[r] - base[r]);
    __syncwarp();
    if (cg == 0) {
#pragma unroll
      for (int r = 0; r < 4; ++r) sum[4 * rg + r] = sum[4 * rg + r] * f[r] + all[r], top[4 * rg + r] = most[r];
    }
    __syncwarp();  // (a row's weights stay within its warp)
    if (f[0] != 1.f || f[1] != 1.f || f[2] != 1.f || f[3] != 1.f) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < DIMS; ++c) acc[r][c] *= f[r];
    }
    auto dim = [&](int c) { return RUN * cg + c / RUN * 64 + c % RUN; };  // this thread's c-th
    if (careful) {
      for (int t = 0; t < KEYS; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float p = ps[t * (ROWS + 4) + 4 * rg + r];
          if (p == 0.f) continue;
#pragma unroll
          for (int c = 0; c < DIMS; ++c) acc[r][c] = fmaf(p, vs[t * STRIDE + dim(c)], acc[r][c]);
        }
    } else {
#pragma unroll 4
      for (int t = 0; t < KEYS; ++t) {
        const float4 p = *reinterpret_cast<const float4*>(ps + t * (ROWS + 4) + 4 * rg);
        float v[DIMS];
#pragma unroll
        for (int c = 0; c < DIMS; c += RUN) {
          if constexpr (RUN == 4) *reinterpret_cast<float4*>(v + c) = *reinterpret_cast<const float4*>(vs + t * STRIDE + dim(c));
          else *reinterpret_cast<float2*>(v + c) = *reinterpret_cast<const float2*>(vs + t * STRIDE + dim(c));
        }
#pragma unroll
        for (int c = 0; c < DIMS; ++c) {
          acc[0][c] = fmaf(p.x, v[c], acc[0][c]), acc[1][c] = fmaf(p.y, v[c], acc[1][c]);
          acc[2][c] = fmaf(p.z, v[c], acc[2][c]), acc[3][c] = fmaf(p.w, v[c], acc[3][c]);
        }
      }
    }
    if (now.tile + 1 < now.tiles && now.left > 1) {
      ++now.tile, --now.left;
      continue;
    }
    // ---- the item's end in this block ----
    __syncthreads();
    const bool whole = !(first && halfway) && now.tile + 1 == now.tiles;
    const size_t slot = 2 * (size_t)blockIdx.x + (first ? 0 : 1);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int mine = 4 * rg + r, row = row0 + mine;
      if (mine >= here) continue;
      if (!whole) {
        const size_t at = slot * ROWS + mine;
        if (cg == 0) a.part_ml[2 * at] = top[mine], a.part_ml[2 * at + 1] = sum[mine];
#pragma unroll
        for (int c = 0; c < DIMS; ++c)
          if (dim(c) < d) a.part_o[at * d + dim(c)] = acc[r][c];
        continue;
      }
      const int token = now.k.first + row / group, head = now.head * group + row % group;
      float l = sum[mine], f = 1.f;
      if (a.sink) {
        const float z = a.sink[head] * LOG2E, base = fmaxf(top[mine], z);
        f = exp2f(top[mine] - base), l = l * f + exp2f(z - base);
      }
      const float unit = l > 0.f || l != l ? f / l : 0.f;
#pragma unroll
      for (int c = 0; c < DIMS; ++c)
        if (dim(c) < d) finish_dim<float>(a, token, head, dim(c), unit == 0.f ? 0.f : acc[r][c] * unit);
    }
    __syncthreads();  // (the next item's rows and queries go where this one's were)
    first = false, entered = true;
    now.next(a, shares);
  }
}

// A warp a (token, head): its pieces in order, the sink, the gate.
template <typename T>
__global__ void __launch_bounds__(THREADS) tree_merge_kernel(const __grid_constant__ TreeAttention a) {
  pdl_wait();
  pdl_launch_dependents();
  const int at = blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (at >= a.tokens * a.nq) return;
  const int token = at / a.nq, head = at % a.nq;
  // The request this token belongs to: the last one that begins at or ahead of it.
  int request = 0, end = a.requests - 1;
  while (request < end) {
    const int mid = (request + end + 1) >> 1;
    if (a.cu_seqlens[mid] <= token) request = mid; else end = mid - 1;
  }
  if (token >= a.cu_seqlens[a.requests]) return;
  const TreeKeys k = tree_keys(a, request);
  const int parts = min(a.parts, (k.total + a.chunk - 1) / a.chunk);
  const size_t step = (size_t)a.tokens * a.nq;
  constexpr int PER = 16;  // dims of a lane, at most
  float sum[PER], l = 0.f, base = -INFINITY;
#pragma unroll
  for (int i = 0; i < PER; ++i) sum[i] = 0.f;
  for (int p0 = 0; p0 < parts; p0 += 32) {  // 32 pieces at a time, a lane each for their offsets and sums
    float ml = -INFINITY, ll = 0.f;
    if (p0 + lane < parts) {
      const float2 x = reinterpret_cast<const float2*>(a.part_ml)[(p0 + lane) * step + at];
      ml = x.x, ll = x.y;
    }
    const float over = fmaxf(base, warp_max(ml)), offset = over == -INFINITY ? 0.f : over, f = exp2f(base - offset), w = exp2f(ml - offset);
    l = l * f + warp_sum(ll * w);
    base = over;
#pragma unroll
    for (int i = 0; i < PER; ++i) sum[i] *= f;
    const int here = min(32, parts - p0);
#pragma unroll 4
    for (int p = 0; p < here; ++p) {
      const float by = __shfl_sync(0xffffffffu, w, p);
      const float* from = a.part_o + ((p0 + p) * step + at) * a.dv;
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (32 * i + lane < a.dv && by != 0.f) sum[i] = fmaf(from[32 * i + lane], by, sum[i]);
    }
  }
  const float sink = a.sink ? a.sink[head] * LOG2E : -INFINITY, over = fmaxf(base, sink), offset = over == -INFINITY ? 0.f : over, f = exp2f(base - offset);
  l = l * f + exp2f(sink - offset);
  const float unit = l > 0.f || l != l ? f / l : 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (32 * i + lane < a.dv) finish_dim<T>(a, token, head, 32 * i + lane, unit == 0.f ? 0.f : sum[i] * unit);
}

template <typename T, int MOST, int KEYS>
int launch_pieces(const TreeAttention& a, int most_nodes, cudaStream_t stream) {
  constexpr int STRIDE = MOST + 4;
  constexpr int bytes = ((ROWS + 2 * KEYS) * STRIDE + KEYS * (ROWS + 4)) * (int)sizeof(float);
  static bool ready[64] = {};
  int device = 0;
  cudaGetDevice(&device);
  if (device < 0 || device >= 64) return (int)cudaErrorInvalidDevice;
  if (!ready[device]) {
    const cudaError_t e = cudaFuncSetAttribute(tree_pieces_kernel<T, MOST, KEYS>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return (int)e;
    ready[device] = true;
  }
  // (The first axis of a grid takes 2^31 - 1 blocks, the others 65,535.)
  const dim3 grid(a.requests * a.nkv, (most_nodes * (a.nq / a.nkv) + ROWS - 1) / ROWS, a.parts);
  launch_pdl(tree_pieces_kernel<T, MOST, KEYS>, grid, dim3(THREADS), bytes, stream, a);
  return OMNIA_LAUNCH_RESULT();
}

template <typename T>
int launch_tree(const TreeAttention& a, int most_nodes, cudaStream_t stream) {
  const int most = a.d > a.dv ? a.d : a.dv;
  if (most <= 64) return launch_pieces<T, 64, 64>(a, most_nodes, stream);
  if (most <= 128) return launch_pieces<T, 128, 64>(a, most_nodes, stream);
  if (most <= 256) return launch_pieces<T, 256, 32>(a, most_nodes, stream);
  return launch_pieces<T, 512, 16>(a, most_nodes, stream);
}

template <int MOST>
int launch_shares32(TreeAttention a, int most_nodes, int blocks, cudaStream_t stream) {
  using S = Shares32<MOST>;
  a.parts = tree_row_tiles(a, most_nodes, ROWS);
  constexpr int bytes = S::FLOATS * (int)sizeof(float);
  static bool ready[64] = {};
  int device = 0;
  cudaGetDevice(&device);
  if (device < 0 || device >= 64) return (int)cudaErrorInvalidDevice;
  if (!ready[device]) {
    const cudaError_t e = cudaFuncSetAttribute(tree_shares32_kernel<MOST>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return (int)e;
    ready[device] = true;
  }
  launch_pdl(tree_shares32_kernel<MOST>, dim3(blocks), dim3(THREADS), bytes, stream, a);
  const int code = OMNIA_LAUNCH_RESULT();
  if (code) return code;
  return tree_join<float, MOST <= 128 ? 128 : 256>(a, {ROWS, S::KEYS, 1, S::EXTRA}, most_nodes, blocks, stream);
}

}  // namespace

extern "C" int omnia_tree_attention(const TreeAttention* a, int most_nodes, int dtype, void* stream) {
  if (a->d < 1 || a->dv < 1 || a->d > 512 || a->dv > 512 || a->nkv < 1 || a->nq % a->nkv || a->requests < 1 ||
      (long long)a->requests * a->nkv > 0x7fffffffLL || a->parts > 65535 || most_nodes < 1 || a->chunk < 1 || a->parts < 1 || a->page_size < 1)
    return (int)cudaErrorInvalidValue;
  OMNIA_DISPATCH_DTYPE(dtype, return launch_tree<T>(*a, most_nodes, (cudaStream_t)stream));
}

extern "C" int omnia_tree_merge(const TreeAttention* a, int dtype, void* stream) {
  if ((uintptr_t)a->part_ml & 7) return (int)cudaErrorInvalidValue;  // (offsets and sums are read in pairs)
  const dim3 grid((a->tokens * a->nq + THREADS / 32 - 1) / (THREADS / 32));
  OMNIA_DISPATCH_DTYPE(dtype, launch_pdl(tree_merge_kernel<T>, grid, dim3(THREADS), 0, (cudaStream_t)stream, *a));
  return OMNIA_LAUNCH_RESULT();
}

// The 32-bit path: keys and values of one width, a multiple of 4 up to 256. `blocks`: what the work is shared out over, with two slots of
// ROWS rows each in part_o and part_ml.
extern "C" int omnia_tree_attention32(const TreeAttention* a, int most_nodes, int blocks, void* stream) {
  if (a->d != a->dv || a->d % 4 || a->d < 4 || a->d > 256 || a->nkv < 1 || a->nkv > 65535 || a->nq % a->nkv || a->requests < 1 ||
      a->requests > TREE_MOST_REQUESTS || most_nodes < 1 || blocks < 1 || a->page_size < 1 || a->page_stride % 4 ||
      (((uintptr_t)a->k_pages | (uintptr_t)a->v_pages) & 15))
    return (int)cudaErrorInvalidValue;
  const cudaStream_t s = (cudaStream_t)stream;
  if (a->d <= 32) return launch_shares32<32>(*a, most_nodes, blocks, s);
  if (a->d <= 64) return launch_shares32<64>(*a, most_nodes, blocks, s);
  if (a->d <= 128) return launch_shares32<128>(*a, most_nodes, blocks, s);
  return launch_shares32<256>(*a, most_nodes, blocks, s);
}
