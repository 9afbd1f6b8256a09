// Attention of trees of drafted tokens for any head sizes (<= 512; keys and values may differ in width), page size and element type, and the
// merge of the pieces that all kernels of such attention leave behind.
//
//   out[i, h] = sigmoid(gate) * sum_k p_k v_k / (sum_k p_k + exp(sink_h)),  p_k = exp(s_k), s_k = scale q_i . k (softcap tanh(s / softcap))
//
// over the keys that node i sees (attention_tree.cuh); a node that sees nothing has zeros.
//
// The rows of a tile are (node, query head of the group) pairs of one key/value head, so that a key fetched is used by all of them. A block
// has a tile of 32 rows and a run of `chunk` keys, which it walks in tiles held in shared memory as float32, with the softmax's
// maximum and sum kept along; products run on the ordinary float32 units, a thread 4 rows x 4 keys and 4 rows x D / 16 dims. With more than one
// chunk a block writes its maximum, sum and unnormalised sums to memory and the merge adds them in the chunks' order, so the
// result does not depend on which block was first.
#include "attention_tree.cuh"

namespace {

constexpr int THREADS = 128, ROWS = 32;
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ bool tid0() { return threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0; }

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
  __shared__ int low[ROWS], node_pos[KEYS], key_of[KEYS];
  __shared__ float top[ROWS], sum[ROWS], factor[ROWS];
  pdl_wait();
  pdl_launch_dependents();
  const int request = blockIdx.z / a.nkv, kvh = blockIdx.z % a.nkv, part = blockIdx.x, group = a.nq / a.nkv;
  const TreeKeys k = tree_keys(a, request);
  if ((k.total > (long long)a.parts * a.chunk || k.count * group > (int)gridDim.y * ROWS) && tid0()) atomicOr(a.err, OMNIA_ERR_WORK);
  const int rows = k.count * group, row0 = blockIdx.y * ROWS, here = min(rows - row0, ROWS);
  if (here <= 0) return;
  const int x0 = part * a.chunk, x1 = min(x0 + a.chunk, k.total);
  if (x0 >= x1 && part > 0) return;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
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
  for (int x = x0; x < x1; x += KEYS) {
    __syncthreads();
    if (tid < KEYS) {
      int key = -1, pos = 0;
      if (x + tid < x1) {
        key = k.key(x + tid);
        const int page = key / a.page_size;
        pos = key < k.held ? key : a.positions[k.first + key - k.held];
        if (page >= a.max_pages || table[page] < 0 || table[page] >= a.num_pages) atomicOr(a.err, OMNIA_ERR_PAGE), key = -1;
      }
      key_of[tid] = key, node_pos[tid] = pos;
    }
    __syncthreads();
    bool odd = false;  // whether a value is no finite number: what a row does not see then stays out of its sums by a test, for 0 x NaN is NaN
    for (int t = warp; t < KEYS; t += THREADS / 32) {
      const int key = key_of[t];
      const T *krow = nullptr, *vrow = nullptr;
      if (key >= 0) {
        const long long page = table[key / a.page_size], off = kvh * a.page_size + key % a.page_size;
        krow = kp + page * a.page_stride + off * a.d, vrow = vp + page * a.page_stride + off * a.dv;
      }
      for (int c = lane; c < MOST; c += 32) {
        ks[t * STRIDE + c] = krow && c < a.d ? to_f32(krow[c]) : 0.f;
        const float v = vrow && c < a.dv ? to_f32(vrow[c]) : 0.f;
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
    const float unit = l > 0.f ? f / l : 0.f;
#pragma unroll
    for (int c = 0; c < DIMS; ++c)
      if (cg + 16 * c < a.dv) finish_dim<T>(a, token, head, cg + 16 * c, acc[r][c] * unit);
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
  float base = a.sink ? a.sink[head] * LOG2E : -INFINITY;
  const size_t step = (size_t)a.tokens * a.nq;
  for (int p = lane; p < parts; p += 32) base = fmaxf(base, a.part_ml[2 * (p * step + at)]);
  base = warp_max(base);
  if (base == -INFINITY) base = 0.f;
  float l = a.sink ? exp2f(a.sink[head] * LOG2E - base) : 0.f;
  for (int p = 0; p < parts; ++p) l += a.part_ml[2 * (p * step + at) + 1] * exp2f(a.part_ml[2 * (p * step + at)] - base);
  const float unit = l > 0.f ? 1.f / l : 0.f;
  for (int c = lane; c < a.dv; c += 32) {
    float v = 0.f;
    for (int p = 0; p < parts; ++p) {
      const float w = exp2f(a.part_ml[2 * (p * step + at)] - base);
      if (w > 0.f) v = fmaf(a.part_o[(p * step + at) * a.dv + c], w, v);
    }
    finish_dim<T>(a, token, head, c, v * unit);
  }
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
  const dim3 grid(a.parts, (most_nodes * (a.nq / a.nkv) + ROWS - 1) / ROWS, a.requests * a.nkv);
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

}  // namespace

extern "C" int omnia_tree_attention(const TreeAttention* a, int most_nodes, int dtype, void* stream) {
  if (a->d < 1 || a->dv < 1 || a->d > 512 || a->dv > 512 || a->nkv < 1 || a->nq % a->nkv || a->requests < 1 || (long long)a->requests * a->nkv > 65535 ||
      most_nodes < 1 || a->chunk < 1 || a->parts < 1 || a->page_size < 1)
    return (int)cudaErrorInvalidValue;
  OMNIA_DISPATCH_DTYPE(dtype, return launch_tree<T>(*a, most_nodes, (cudaStream_t)stream));
}

extern "C" int omnia_tree_merge(const TreeAttention* a, int dtype, void* stream) {
  const dim3 grid((a->tokens * a->nq + THREADS / 32 - 1) / (THREADS / 32));
  OMNIA_DISPATCH_DTYPE(dtype, launch_pdl(tree_merge_kernel<T>, grid, dim3(THREADS), 0, (cudaStream_t)stream, *a));
  return OMNIA_LAUNCH_RESULT();
}
