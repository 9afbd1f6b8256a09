// Paged attention of single tokens whose requests share their first positions, for any element type, head sizes (<= 512,
// keys and values may differ in width), group and page size: the kernels of the 32-bit path, and of bfloat16 sizes that have no
// tensor-core decode kernel; and the list of what is shared, which all kernels for shared positions read.
//
// Softmax attention over any cut of a row's keys comes together from each piece's maximum m, sum l = sum e^(z - m) and
// accumulator o = sum e^(z - m) v:  m = max m_i,  l = sum l_i e^(m_i - m),  o = sum o_i e^(m_i - m),  and the row's answer is
// o / l (l + e^(sink - m) under a sink). So the positions that a group of requests shares are one piece, or several, attended
// to by all of the group's rows at once: their keys and values are read once for the group and not once a request. What a request holds
// of its own makes more pieces. Everything is held in float32.
//
// Pieces are written as [requests, heads, places, width] (m in log2 units), a request's shared ones first, and a kernel of a
// block per request and head puts them together, adds the sink, takes the difference of two maps or the gate.
//
// A block of four warps owns up to 32 rows (request, query head) of one key/value head and walks its keys in tiles of 32: a
// warp has eight of the rows, a lane scores one key for them and then owns output dims lane, lane + 32, ... Four blocks an SM.
//
// Floor: the shared keys and values once, each request's own once. What bounds it is neither these nor its multiplications but a tile's
// chain (table, rows, scores, weights), which four blocks an SM fill in part: 12 requests of 1,001 shared positions and up to 65 of
// their own, 8/1 heads of 24 in 32 bits, 17 us (0.3 MB), where each request for itself takes 299. With a lookup of the table and a trip to
// memory a key 48, without these 37; the rest was rows one after the other, and a merge a load at a time.
#include "attention_shared.cuh"

namespace {

constexpr int ROWS = 32, WARPS = 4, PER_WARP = ROWS / WARPS, TILE = 32;
constexpr float LOG2E = 1.4426950408889634f;

}  // namespace

namespace {

// A tile of up to 32 keys for N of a warp's rows (every WARPS-th row of the block), all at once and without a branch between them, so that their
// reductions overlap. Rows beyond the block's hold zeros and are written nowhere.
template <int N, int ACC>
__device__ __forceinline__ void attend_rows(const float* q, const float* ks, const float* vs, int stride, int width4, int dv, int keys, bool capped,
                                            float pre, float cap, float* m, float* l, float (*acc)[ACC]) {
  const int lane = threadIdx.x & 31;
  float s[N];
#pragma unroll
  for (int x = 0; x < N; ++x) s[x] = 0.f;
  const float4* k4 = reinterpret_cast<const float4*>(ks + lane * stride);
#pragma unroll 2
  for (int c = 0; c < width4; ++c) {
    const float4 k = k4[c];
#pragma unroll
    for (int x = 0; x < N; ++x) {
      const float4 v = reinterpret_cast<const float4*>(q + WARPS * x * stride)[c];
      s[x] = fmaf(v.x, k.x, fmaf(v.y, k.y, fmaf(v.z, k.z, fmaf(v.w, k.w, s[x]))));
    }
  }
  float top[N], sum[N];
#pragma unroll
  for (int x = 0; x < N; ++x) {
    s[x] = capped ? cap * tanhf(s[x] * pre) : s[x] * pre;
    if (lane >= keys) s[x] = -INFINITY;
    top[x] = s[x];
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1)
#pragma unroll
    for (int x = 0; x < N; ++x) top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], off));
#pragma unroll
  for (int x = 0; x < N; ++x) {
    top[x] = fmaxf(m[x], top[x]);
    const float base = top[x] == -INFINITY ? 0.f : top[x];
    const float alpha = m[x] == -INFINITY ? 0.f : exp2f(m[x] - base);
    s[x] = sum[x] = exp2f(s[x] - base);
    m[x] = top[x], l[x] *= alpha;
#pragma unroll
    for (int k = 0; k < ACC; ++k) acc[x][k] *= alpha;
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1)
#pragma unroll
    for (int x = 0; x < N; ++x) sum[x] += __shfl_xor_sync(0xffffffffu, sum[x], off);
#pragma unroll
  for (int x = 0; x < N; ++x) l[x] += sum[x];
#pragma unroll 4
  for (int k = 0; k < TILE; ++k) {  // (keys past the last have no weight, and zeros for values)
    float v[ACC];
#pragma unroll
    for (int i = 0; i < ACC; ++i) v[i] = lane + 32 * i < dv ? vs[k * dv + lane + 32 * i] : 0.f;
#pragma unroll
    for (int x = 0; x < N; ++x) {
      const float p = __shfl_sync(0xffffffffu, s[x], k);
#pragma unroll
      for (int i = 0; i < ACC; ++i) acc[x][i] = fmaf(p, v[i], acc[x][i]);
    }
  }
}

template <typename T, int MOST>
__global__ void __launch_bounds__(32 * WARPS)
shared_pieces_kernel(const __grid_constant__ SharedAttention a) {
  constexpr int ACC = MOST / 32, AT_ONCE = ACC < 4 ? ACC : 4;
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int group = a.nq / a.nkv, width4 = (a.d + 3) / 4;
  const int stride = 4 * width4 + ((width4 & 1) ? 0 : 4);  // 4 modulo 8 floats: eight lanes' 16 bytes lie in different banks
  const int *starts = a.plan, *parts = starts + a.requests, *members = parts + a.requests;
  int table_of, first_member, row0, rows, kvh, lo, hi, part;
  if ((int)blockIdx.x < a.items) {
    const int* item = members + a.members + SHARED_ITEM_INTS * blockIdx.x;
    table_of = item[0], first_member = item[1], row0 = item[2], rows = item[3], kvh = item[4], lo = item[5], hi = item[6], part = item[7];
  } else {
    // A chunk of what a request holds of its own.
    int at = blockIdx.x - a.items;
    const int chunk = at % a.max_chunks;
    at /= a.max_chunks;
    const int blocks = (group + ROWS - 1) / ROWS;
    row0 = at % blocks * ROWS;
    at /= blocks;
    kvh = at % a.nkv;
    table_of = at / a.nkv;
    first_member = -1;
    rows = min(ROWS, group - row0);
    lo = starts[table_of] + chunk * a.chunk_keys, hi = min(lo + a.chunk_keys, a.seq_lens[table_of]);
    part = parts[table_of] + chunk;
  }
  if (rows < 1 || lo >= hi) return;

  extern __shared__ __align__(16) float smem[];
  float* qs = smem;                    // [ROWS][stride]
  float* ks = qs + ROWS * stride;      // [TILE][stride]
  float* vs = ks + TILE * stride;      // [TILE][dv]
  auto place = [&](int r, int& request, int& head) {
    const int row = row0 + r;
    request = first_member < 0 ? table_of : members[first_member + row / group];
    head = kvh * group + row % group;
  };
  const T* q = (const T*)a.q;
  for (int i = tid; i < ROWS * stride; i += 32 * WARPS) {
    const int r = i / stride, c = i - r * stride;
    float v = 0.f;
    if (r < rows && c < a.d) {
      int request, head;
      place(r, request, head);
      v = to_f32(q[((size_t)a.cu_seqlens[request] * a.nq + head) * a.d + c]);
    }
    qs[i] = v;
  }
  for (int i = tid; i < TILE * stride; i += 32 * WARPS) ks[i] = 0.f;  // the dims beyond d stay zero
  float m[PER_WARP], l[PER_WARP], acc[PER_WARP][ACC];
#pragma unroll
  for (int x = 0; x < PER_WARP; ++x) {
    m[x] = -INFINITY, l[x] = 0.f;
#pragma unroll
    for (int k = 0; k < ACC; ++k) acc[x][k] = 0.f;
  }
  const int* table = a.block_table + (size_t)table_of * a.max_pages;
  const T *k_pages = (const T*)a.k_pages, *v_pages = (const T*)a.v_pages;
  const float pre = a.softcap > 0.f ? a.scale / a.softcap : a.scale * LOG2E, cap = a.softcap * LOG2E;
  for (int key0 = lo; key0 < hi; key0 += TILE) {
    __syncthreads();  // the tile before has been read
    const int keys = min(TILE, hi - key0);
    // A lane looks a key's page up; then a warp brings every fourth key, the loads of 128 columns of all of its keys and values on their way
    // together. Rows past the last key hold zeros, whatever the cache has there.
    int page = -1;
    if (lane < keys) {
      page = table[(key0 + lane) / a.page_size];
      if (page < 0 || page >= a.num_pages) page = -1;
    }
    if (warp == 0 && __any_sync(0xffffffffu, lane < keys && page < 0) && lane == 0) atomicOr(a.err, OMNIA_ERR_PAGE);
    const T *k_rows[PER_WARP], *v_rows[PER_WARP];
#pragma unroll
    for (int x = 0; x < PER_WARP; ++x) {
      const int k = warp + WARPS * x, from = __shfl_sync(0xffffffffu, page, k);
      const long long at = (long long)from * a.page_stride;
      const int off = kvh * a.page_size + (key0 + k) % a.page_size;
      k_rows[x] = from < 0 ? nullptr : k_pages + at + (long long)off * a.d;
      v_rows[x] = from < 0 ? nullptr : v_pages + at + (long long)off * a.dv;
    }
#pragma unroll 1
    for (int c0 = lane; c0 < MOST; c0 += 32 * AT_ONCE) {
      T k[PER_WARP][AT_ONCE], v[PER_WARP][AT_ONCE];
#pragma unroll
      for (int x = 0; x < PER_WARP; ++x)
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
          const int c = c0 + 32 * i;
          k[x][i] = k_rows[x] != nullptr && c < a.d ? k_rows[x][c] : from_f32<T>(0.f);
          v[x][i] = v_rows[x] != nullptr && c < a.dv ? v_rows[x][c] : from_f32<T>(0.f);
        }
#pragma unroll
      for (int x = 0; x < PER_WARP; ++x)
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
          const int c = c0 + 32 * i;
          if (c < a.d) ks[(warp + WARPS * x) * stride + c] = to_f32(k[x][i]);
          if (c < a.dv) vs[(warp + WARPS * x) * a.dv + c] = to_f32(v[x][i]);
        }
    }
    __syncthreads();
    if (rows > 2 * WARPS)
      attend_rows<PER_WARP, ACC>(qs + warp * stride, ks, vs, stride, width4, a.dv, keys, a.softcap > 0.f, pre, cap, m, l, acc);
    else
      attend_rows<2, ACC>(qs + warp * stride, ks, vs, stride, width4, a.dv, keys, a.softcap > 0.f, pre, cap, m, l, acc);
  }
  const int places = a.max_parts + a.max_chunks;
#pragma unroll
  for (int x = 0; x < PER_WARP; ++x) {
    const int r = warp + WARPS * x;
    if (r >= rows) break;
    int request, head;
    place(r, request, head);
    const size_t at = ((size_t)request * a.nq + head) * places + part;
#pragma unroll
    for (int i = 0; i < ACC; ++i)
      if (lane + 32 * i < a.dv) a.part_o[at * a.dv + lane + 32 * i] = acc[x][i];
    if (lane == 0) a.part_ml[2 * at] = m[x], a.part_ml[2 * at + 1] = l[x];
  }
}

// grid (heads that come out, requests), 128 threads: a request's pieces put together in ascending order.
// What a request holds of its own was cut from its first such position on or (`fixed`: by the decode kernel) at multiples of chunk_keys.
template <typename T>
__global__ void __launch_bounds__(128)
shared_merge_kernel(const __grid_constant__ SharedAttention a, int fixed) {
  __shared__ float scratch[33];
  // The kernel before this one lets it begin only after its own wait for whatever came before, so lengths and list are there.
  const int request = blockIdx.y, tid = threadIdx.x, length = a.seq_lens[request], start = a.plan[request], parts = a.plan[a.requests + request];
  const size_t token = (size_t)a.cu_seqlens[request];
  pdl_wait();
  pdl_launch_dependents();
  if (length < 1) return;
  const int own = length - (fixed ? start / a.chunk_keys * a.chunk_keys : start);
  // More than the step was laid out for, or no more than is shared.
  if ((own > a.max_chunks * (long long)a.chunk_keys || length <= start) && blockIdx.x == 0 && tid == 0) atomicOr(a.err, OMNIA_ERR_WORK);
  const int count = min(parts, a.max_parts) + max(0, min((own + a.chunk_keys - 1) / a.chunk_keys, a.max_chunks));
  const int places = a.max_parts + a.max_chunks;
  constexpr int PER_THREAD = 4;  // widths of at most 512
  float map[2][PER_THREAD];
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if (which >= a.maps) break;
    const int head = blockIdx.x * a.maps + which;
    const size_t at = ((size_t)request * a.nq + head) * places;
    const float *ml = a.part_ml + 2 * at, *o = a.part_o + at * a.dv;
    float top = -INFINITY, total = 0.f;
#pragma unroll
    for (int v = 0; v < PER_THREAD; ++v) map[which][v] = 0.f;
    // Rounds of 32 pieces: a lane has one's maximum and sum; then sixteen accumulators on their way at a time.
    for (int done = 0; done < count; done += 32) {
      const int some = min(32, count - done), lane = tid & 31;
      const float m = lane < some ? __ldcg(ml + 2 * (done + lane)) : -INFINITY, l = lane < some ? __ldcg(ml + 2 * (done + lane) + 1) : 0.f;
      const float now = fmaxf(top, warp_max(m)), keep = top == -INFINITY ? 0.f : exp2f(top - now);
      const float w = m == -INFINITY ? 0.f : exp2f(m - now);
      total = total * keep + warp_sum(l * w);
#pragma unroll
      for (int v = 0; v < PER_THREAD; ++v) map[which][v] *= keep;
      top = now;
      for (int i0 = 0; i0 < some; i0 += 16) {
#pragma unroll
        for (int v = 0; v < PER_THREAD; ++v) {
          if (128 * v >= a.dv) break;
          const int dim = tid + 128 * v;
          float x[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] = i0 + i < some && dim < a.dv ? __ldcg(o + (size_t)(done + i0 + i) * a.dv + dim) : 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) map[which][v] = fmaf(x[i], __shfl_sync(0xffffffffu, w, i0 + i), map[which][v]);
        }
      }
    }
    if (a.sink != nullptr && top != -INFINITY) total += exp2f(a.sink[head] * LOG2E - top);
    const float inv = total > 0.f ? 1.f / total : 0.f;
#pragma unroll
    for (int v = 0; v < PER_THREAD; ++v) map[which][v] *= inv;
  }
  T* out = (T*)a.out;
  if (a.maps == 2) {
    float ss = 0.f;
#pragma unroll
    for (int v = 0; v < PER_THREAD; ++v) {
      map[0][v] = tid + 128 * v < a.difference.dv ? map[0][v] - a.difference.lambda * map[1][v] : 0.f;
      ss += map[0][v] * map[0][v];
    }
    const float f = rsqrtf(block_sum(ss, scratch) / (float)a.difference.dv + a.difference.eps) * a.difference.factor;
    T* row = out + (token * (a.nq / 2) + blockIdx.x) * a.difference.dv;
#pragma unroll
    for (int v = 0; v < PER_THREAD; ++v)
      if (tid + 128 * v < a.difference.dv) row[tid + 128 * v] = from_f32<T>(map[0][v] * f);
    return;
  }
  const T* gate = a.gate ? (const T*)a.gate + token * a.gate_stride + (size_t)blockIdx.x * a.dv : nullptr;
#pragma unroll
  for (int v = 0; v < PER_THREAD; ++v) {
    const int dim = tid + 128 * v;
    if (dim >= a.dv) break;
    float y = map[0][v];
    if (gate) y *= 1.f / (1.f + expf(-to_f32(gate[dim])));
    out[(token * a.nq + blockIdx.x) * a.dv + dim] = from_f32<T>(y);
  }
}

template <typename T, int MOST>
int launch_pieces(const SharedAttention& a, long long blocks, size_t smem, cudaStream_t stream) {
  static bool configured[64] = {};
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return (int)cudaErrorInvalidDevice;
  if (!configured[device]) {
    const cudaError_t e = cudaFuncSetAttribute(shared_pieces_kernel<T, MOST>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
    if (e != cudaSuccess) return (int)e;
    configured[device] = true;
  }
  launch_pdl(shared_pieces_kernel<T, MOST>, dim3((unsigned)blocks), 32 * WARPS, smem, stream, a);
  return OMNIA_LAUNCH_RESULT();
}

}  // namespace

// The pieces that the decode kernel has left (omnia_attention_decode_shared with `rows`), of any width.
extern "C" int omnia_shared_merge(const SharedAttention* given, int dtype, cudaStream_t stream) {
  const SharedAttention a = *given;
  if (a.requests == 0) return 0;
  if (a.requests < 0 || a.requests > 65535 || a.nkv < 1 || a.nq < 1 || a.nq % a.nkv || a.dv < 1 || a.dv > 512 || a.max_parts < 0 || a.max_chunks < 0 ||
      a.chunk_keys < 1 || (a.maps != 1 && a.maps != 2) ||
      (a.maps == 2 && (a.nq % 2 || a.gate || a.sink || a.difference.dv < 1 || a.difference.dv > a.dv)))
    return (int)cudaErrorInvalidValue;
  OMNIA_DISPATCH_DTYPE(dtype, launch_pdl(shared_merge_kernel<T>, dim3(a.nq / a.maps, a.requests), 128, 0, stream, a, 1));
  return OMNIA_LAUNCH_RESULT();
}

extern "C" int omnia_shared_attention(const SharedAttention* given, int dtype, cudaStream_t stream) {
  const SharedAttention a = *given;
  if (a.requests == 0) return 0;
  if (a.requests < 0 || a.requests > 65535 || a.members < 0 || a.items < 0 || a.nkv < 1 || a.nq < 1 || a.nq % a.nkv || a.d < 1 || a.d > 512 ||
      a.dv < 1 || a.dv > 512 || a.page_size < 1 || a.max_pages < 1 || a.num_pages < 1 || a.max_parts < 0 || a.max_chunks < 0 ||
      a.chunk_keys < 1 || a.softcap < 0.f || (a.maps != 1 && a.maps != 2) ||
      (a.maps == 2 && (a.nq % 2 || a.gate || a.sink || a.difference.dv < 1 || a.difference.dv > a.dv)))
    return (int)cudaErrorInvalidValue;
  const int group = a.nq / a.nkv, width4 = (a.d + 3) / 4, stride = 4 * width4 + ((width4 & 1) ? 0 : 4);
  const long long blocks = a.items + (long long)a.requests * a.nkv * ((group + ROWS - 1) / ROWS) * a.max_chunks;
  if (blocks > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
  const size_t smem = (size_t)((ROWS + TILE) * stride + TILE * a.dv) * sizeof(float);
  const int most = a.d > a.dv ? a.d : a.dv;
  OMNIA_DISPATCH_DTYPE(dtype, {
    if (blocks > 0) {
      const int code = most <= 64 ? launch_pieces<T, 64>(a, blocks, smem, stream) : most <= 128 ? launch_pieces<T, 128>(a, blocks, smem, stream)
                     : most <= 256 ? launch_pieces<T, 256>(a, blocks, smem, stream) : launch_pieces<T, 512>(a, blocks, smem, stream);
      if (code != 0) return code;
    }
    launch_pdl(shared_merge_kernel<T>, dim3(a.nq / a.maps, a.requests), 128, 0, stream, a, 0);
  });
  return OMNIA_LAUNCH_RESULT();
}
