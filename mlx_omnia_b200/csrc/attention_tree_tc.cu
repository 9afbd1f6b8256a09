// Attention of trees of drafted tokens in bfloat16 on the tensor cores (mma.sync m16n8k16, float32 sums and softmax), for requests that bring few rows.
// Compiled for one head size:
//   -DHEAD_DIM=d   (a multiple of 8, at most 256; rows are zero-padded to a multiple of 16; keys and values of equal width)
//
// Rows of a tile are (node, query head of the group) pairs of one request and key/value head, 16, 32 or 64 of them; four warps share a
// tile of 64 keys, each with sixteen of the rows and all, half or a quarter of the keys, with a softmax state of its own; the states are brought
// together when an item ends. Keys and values come by cp.async, row by row through the block table, so any page size works, three tiles deep, and
// the loads run on across the items of a block's share (TreeShares).
//
// Floor: a request's keys and values once, 4 D bytes a position and key/value head. mma.sync gets to some 155 TFLOP/s here, so 16 rows to a key are what the
// memory's rate allows; that is why tiles of 16 rows share the keys out among the warps, and why the tcgen05 kernel takes over above them. 16 / 8 heads of 128:
// one request of 500 positions with 5 tokens 11.1 us (2.1 MB: 0.3 us; shares known after 2, a first tile there after 4.6, the sums at 7.7, then the join), of 4,000
// 19.4, four of 1,000 14.4; 8 of 20,000 with 8 tokens 141 us, 4.7 TB/s. Scores and sums are float32; queries as they came, weights rounded to bfloat16
// for the product with the values as that product takes them (up to 2^-8 of a weight; the sum of weights is of what was not rounded).
//
// What a row does not see has no weight, whatever it holds: scores are replaced before the softmax, and where a tile has something that only some
// rows see (nodes, the edge of a window) its values are looked through for ones that are no numbers, and if there are any, summed by hand.
#include "attention_tree.cuh"

#ifndef HEAD_DIM
#define HEAD_DIM 128
#endif

namespace {

typedef __nv_bfloat16 bf16;

constexpr int D = HEAD_DIM;
static_assert(D % 8 == 0 && D >= 8 && D <= 256, "head size must be a multiple of 8, at most 256");
constexpr int DP = (D + 15) / 16 * 16, ROW = DP + 8;  // padded head size; shared-memory row stride (elements): odd in 16-byte units
constexpr int CH = D / 8, KSTEPS = DP / 16, NT_O = DP / 8;
constexpr int KEYS = 64, WARPS = 4, THREADS = 32 * WARPS, WARP_LOADS = KEYS / WARPS;  // keys whose rows a warp fetches
constexpr int STAGES = D <= 128 ? 3 : 2;
constexpr int EXTRA = 3;                              // tiles that an item's beginning and end cost
constexpr int STAGE = 2 * KEYS * ROW;                 // elements: keys, then values
constexpr float LOG2E = 1.4426950408889634f;
constexpr float RESCALE_STEP = 8.f;  // log2 of how far a row's maximum may outgrow its exponent's offset

__device__ __forceinline__ void cp_async16(void* smem, const void* gmem, bool valid) {
  const unsigned s = (unsigned)__cvta_generic_to_shared(smem);
  const int bytes = valid ? 16 : 0;  // 0 source bytes: the 16 destination bytes are zero-filled
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(s), "l"(gmem), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4(unsigned* r, const bf16* p) {
  const unsigned s = (unsigned)__cvta_generic_to_shared(p);
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(s) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(unsigned* r, const bf16* p) {
  const unsigned s = (unsigned)__cvta_generic_to_shared(p);
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(s) : "memory");
}
__device__ __forceinline__ void mma_bf16(float* c, const unsigned* a, unsigned b0, unsigned b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float fast_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ unsigned pack(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<unsigned*>(&v);
}
__device__ __forceinline__ long long shfl64(long long v, int lane) { return __shfl_sync(0xffffffffu, v, lane); }

}  // namespace

// WR: warps side by side over the rows (a tile has 16 WR); the others share the keys.
template <int WR>
__global__ void __launch_bounds__(THREADS, D <= 128 ? 2 : 1) tree_shares_kernel(const __grid_constant__ TreeAttention a) {
  constexpr int WK = WARPS / WR, KW = KEYS / WK, NT_S = KW / 8, ROWS = 16 * WR, HALF = NT_O > 8 ? (NT_O + 1) / 2 : NT_O;
  extern __shared__ __align__(16) unsigned char raw[];
  bf16* stages = reinterpret_cast<bf16*>(raw);
  float* spare = reinterpret_cast<float*>(stages + STAGES * STAGE);  // [WR][16][8 HALF + 4], one warp's sums on their way to another
  constexpr int SPARE = 8 * HALF + 4;
  float* spare_ml = spare + WR * 16 * SPARE;                         // [WR][16][2]
  __shared__ long long sums[WARPS];
  long long* ends = reinterpret_cast<long long*>(raw);               // (where the stages are to be)
  static_assert(STAGES * STAGE * sizeof(bf16) >= TREE_MOST_REQUESTS * sizeof(long long), "the requests' ends lie in the stages");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, wr = warp % WR, wk = warp / WR, g = lane >> 2, t4 = lane & 3;
  pdl_wait();
  pdl_launch_dependents();
  const TreeShares shares = {ROWS, KEYS, 1, EXTRA};
  const long long total = shares.lay_out(a, ends, sums);
  const long long blocks = min((long long)gridDim.x, total);  // (a block more than there are tiles would leave its slots unwritten)
  if (blockIdx.x >= blocks) return;
  const long long t0 = total * blockIdx.x / blocks, upto = total * (blockIdx.x + 1) / blocks;
  const int group = a.nq / a.nkv;
  const bf16 *kp = static_cast<const bf16*>(a.k_pages), *vp = static_cast<const bf16*>(a.v_pages);
  const long long apart = vp - kp;

  // ---- loads: lane l < 16 knows where the l-th row of its warp's share of a tile lies ------------------------------------------------
  TreePlace ahead;
  ahead.find(a, shares, ends, t0, (int)(upto - t0));
  if (ahead.left == 0) return;
  TreePlace now = ahead;
  OMNIA_TRACE_BLOCK(2);  // the shares are known
  __syncthreads();
  if constexpr (D != DP) {  // the columns beyond a row: no load writes them
    for (int i = tid; i < STAGES * 2 * KEYS; i += THREADS) *reinterpret_cast<uint4*>(stages + i * ROW + D) = make_uint4(0u, 0u, 0u, 0u);
  }
  int load_stage = 0;
  auto where = [&]() -> long long {  // of this lane's key of the place `ahead`: elements from the pages' beginning; -1: none
    const int x = ahead.tile * KEYS + warp * WARP_LOADS + lane;
    if (lane >= WARP_LOADS || x >= ahead.k.total) return -1;
    const int key = ahead.k.key(x), at = key / a.page_size;
    const int page = at < a.max_pages ? a.block_table[(size_t)ahead.request * a.max_pages + at] : -1;
    if (page < 0 || page >= a.num_pages) {
      atomicOr(a.err, OMNIA_ERR_PAGE);
      return -1;
    }
    return page * a.page_stride + (long long)(ahead.head * a.page_size + key % a.page_size) * D;
  };
  long long row_at = where();
  auto fetch = [&]() {  // the tile at `ahead`, into the next stage; then on
    if (ahead.left > 0) {
      bf16* k_s = stages + load_stage * STAGE + warp * WARP_LOADS * ROW;
      if (++load_stage == STAGES) load_stage = 0;
      bf16* v_s = k_s + KEYS * ROW;
      constexpr int PIECES = WARP_LOADS * CH;
#pragma unroll
      for (int i0 = 0; i0 < PIECES; i0 += 32) {
        const int i = i0 + lane, row = min(i / CH, WARP_LOADS - 1), c = i % CH;
        const long long from = shfl64(row_at, row);
        if (PIECES % 32 == 0 || i < PIECES) {
          const bf16* at = kp + (from < 0 ? 0 : from) + c * 8;
          cp_async16(k_s + row * ROW + c * 8, at, from >= 0);
          cp_async16(v_s + row * ROW + c * 8, at + apart, from >= 0);
        }
      }
      ahead.next(a, shares);
      if (ahead.left > 0) row_at = where();
    }
    cp_async_commit();
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) fetch();

  const bool capped = a.softcap > 0.f;
  // Scores keep the sign that they are compared by: a scale below zero turns the queries' signs instead. (A scale of zero is float32's least number: what a
  // row does not see is -infinity ahead of it, which zero would make no number.)
  const float size = fabsf(a.scale), cap = a.softcap * LOG2E, twice = capped ? 2.f * size / a.softcap * LOG2E : 0.f, unit = capped ? 1.f : size == 0.f ? 1.17549435e-38f : size * LOG2E;
  const unsigned turn = a.scale < 0.f ? 0x80008000u : 0u;
  unsigned qf[KSTEPS][4];
  float o[NT_O][4], m[2], l[2];
  int node[2], low[2];
  bool first = true, entered = true;
  int stage = 0;
  const bool halfway = now.tile > 0;  // whether the first item began in another block
  while (now.left > 0) {
    const int rows = now.k.count * group, row0 = now.row_tile * ROWS + 16 * wr;
    if (entered) {
      if (tid == 0 && now.tile == 0) tree_note(a, total, blocks, upto, now, first);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = row0 + g + 8 * h;
        node[h] = row < rows ? row / group : -1;
        low[h] = node[h] >= 0 ? tree_low(a, a.positions[now.k.first + node[h]]) : 0;
        m[h] = -INFINITY, l[h] = 0.f;
        const bf16* q = static_cast<const bf16*>(a.q) + ((size_t)(now.k.first + max(node[h], 0)) * a.nq + now.head * group + row % group) * D;
#pragma unroll
        for (int s = 0; s < KSTEPS; ++s) {
          const int c = 16 * s + 2 * t4;
          qf[s][h] = node[h] >= 0 && c < D ? *reinterpret_cast<const unsigned*>(q + c) ^ turn : 0u;
          qf[s][h + 2] = node[h] >= 0 && c + 8 < D ? *reinterpret_cast<const unsigned*>(q + c + 8) ^ turn : 0u;
        }
      }
#pragma unroll
      for (int i = 0; i < NT_O; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
      entered = false;
    }
    cp_async_wait<STAGES - 2>();
    __syncthreads();
    if (first) OMNIA_TRACE_BLOCK(4);  // a first tile is there
    fetch();
    const bf16* k_s = stages + stage * STAGE + wk * KW * ROW;
    if (++stage == STAGES) stage = 0;
    const bf16* v_s = k_s + KEYS * ROW;
    float s[NT_S][4];
#pragma unroll
    for (int i = 0; i < NT_S; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KSTEPS; ++ks)
#pragma unroll
      for (int i = 0; i < NT_S; i += 2) {
        unsigned b[4];
        ldmatrix_x4(b, k_s + (i * 8 + (lane & 7) + ((lane >> 4) << 3)) * ROW + ks * 16 + ((lane >> 3) & 1) * 8);
        mma_bf16(s[i], qf[ks], b[0], b[1]);
        mma_bf16(s[i + 1], qf[ks], b[2], b[3]);
      }
    const int x0 = now.tile * KEYS + wk * KW;
    if (capped) {  // in log2 units (a score that is infinite has the cap, of its sign: c tanh(x) = c - 2 c / (1 + e^2x))
#pragma unroll
      for (int i = 0; i < NT_S; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = fmaf(-2.f * cap, fast_rcp(1.f + fast_exp2(s[i][j] * twice)), cap);
    }
    // Whether every row sees every key of these.
    const int last_key = now.k.key(min(x0 + KW, now.k.total) - 1);
    const bool clear = x0 + KW <= now.k.total && last_key < now.k.held && x0 >= now.k.kept &&
                       now.k.key(x0) >= tree_low(a, now.k.held + now.k.count - 1);
    if (!clear) {
#pragma unroll
      for (int i = 0; i < NT_S; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int x = x0 + 8 * i + 2 * t4 + j;
          int pos = 0, which = -1;
          const bool real = x < now.k.total;
          if (real) {
            pos = now.k.key(x);
            if (pos >= now.k.held) which = pos - now.k.held, pos = a.positions[now.k.first + which];
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            bool seen = real && node[h] >= 0 && (pos >= low[h] || (a.window > 0 && pos < a.keep));
            if (seen && which >= 0)
              seen = ((unsigned)a.ancestors[(size_t)(now.k.first + node[h]) * a.words + (which >> 5)] >> (which & 31)) & 1u;
            if (!seen) s[i][2 * h + j] = -INFINITY;
          }
        }
    }
    unsigned pf[NT_S / 2][4];
    float p[NT_S][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < NT_S; ++i) top = fmaxf(top, fmaxf(s[i][2 * h], s[i][2 * h + 1]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      top *= unit;
      // The offset follows a row's maximum lazily: what was summed is brought to a new one only when the scores have outgrown the old.
      if (top > m[h]) {
        if (m[h] == -INFINITY) {
          m[h] = top;  // (nothing was summed yet)
        } else if (top - m[h] > RESCALE_STEP) {
          const float f = fast_exp2(m[h] - top);
          m[h] = top, l[h] *= f;
#pragma unroll
          for (int i = 0; i < NT_O; ++i) o[i][2 * h] *= f, o[i][2 * h + 1] *= f;
        }
      }
      const float base = m[h] == -INFINITY ? 0.f : m[h];
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < NT_S; ++i) {
        p[i][2 * h] = fast_exp2(fmaf(s[i][2 * h], unit, -base)), p[i][2 * h + 1] = fast_exp2(fmaf(s[i][2 * h + 1], unit, -base));
        sum += p[i][2 * h] + p[i][2 * h + 1];
      }
      l[h] += sum;  // (of this lane's keys)
      // Weights are rounded to bfloat16 for their product with the values, the sum is of what was not.
#pragma unroll
      for (int i = 0; i < NT_S; i += 2) {
        pf[i / 2][h] = pack(p[i][2 * h], p[i][2 * h + 1]);
        pf[i / 2][h + 2] = pack(p[i + 1][2 * h], p[i + 1][2 * h + 1]);
      }
    }
    bool odd = false;
    if (!clear) {
#pragma unroll 1
      for (int i = lane; i < KW * CH; i += 32) {
        const uint4 v = *reinterpret_cast<const uint4*>(v_s + i / CH * ROW + i % CH * 8);
        for (unsigned w : {v.x, v.y, v.z, v.w}) odd |= (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
      }
      odd = __any_sync(0xffffffffu, odd);
    }
    if (odd) {
#pragma unroll
      for (int i = 0; i < NT_S; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {  // the key that the lane c of a row has at i, j
            const float p0 = __shfl_sync(0xffffffffu, p[i][j], (lane & ~3) | c), p1 = __shfl_sync(0xffffffffu, p[i][2 + j], (lane & ~3) | c);
            const bf16* v = v_s + (8 * i + 2 * c + j) * ROW;
#pragma unroll
            for (int n = 0; n < NT_O; ++n) {
              const float v0 = __bfloat162float(v[8 * n + 2 * t4]), v1 = __bfloat162float(v[8 * n + 2 * t4 + 1]);
              if (p0 != 0.f) o[n][0] = fmaf(p0, v0, o[n][0]), o[n][1] = fmaf(p0, v1, o[n][1]);
              if (p1 != 0.f) o[n][2] = fmaf(p1, v0, o[n][2]), o[n][3] = fmaf(p1, v1, o[n][3]);
            }
          }
    } else {
#pragma unroll
      for (int ks = 0; ks < NT_S / 2; ++ks)
#pragma unroll
        for (int n = 0; n < NT_O; n += 2) {
          unsigned b[4];
          ldmatrix_x4_trans(b, v_s + (ks * 16 + (lane & 15)) * ROW + n * 8 + ((lane >> 4) << 3));
          mma_bf16(o[n], pf[ks], b[0], b[1]);
          mma_bf16(o[n + 1], pf[ks], b[2], b[3]);
        }
    }
    if (now.tile + 1 < now.tiles && now.left > 1) {
      ++now.tile, --now.left;
      continue;
    }
    OMNIA_TRACE_BLOCK(5);  // an item's last product
    // ---- the item's end in this block: the warps that shared the keys, then the slot or the answer ------------------------------------
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    }
#pragma unroll 1
    for (int giver = WK - 1; giver > 0; --giver) {
      float mine[2], other[2];
#pragma unroll
      for (int n0 = 0; n0 < NT_O; n0 += HALF) {
        if (wk == giver) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float* to = spare + (wr * 16 + g + 8 * h) * SPARE;
#pragma unroll
            for (int n = 0; n < HALF; ++n)
              if (n0 + n < NT_O) *reinterpret_cast<float2*>(to + 8 * n + 2 * t4) = make_float2(o[n0 + n][2 * h], o[n0 + n][2 * h + 1]);
            if (n0 == 0 && t4 == 0) spare_ml[(wr * 16 + g + 8 * h) * 2] = m[h], spare_ml[(wr * 16 + g + 8 * h) * 2 + 1] = l[h];
          }
        }
        __syncthreads();
        if (wk == giver - 1) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float* from = spare + (wr * 16 + g + 8 * h) * SPARE;
            if (n0 == 0) {
              const float om = spare_ml[(wr * 16 + g + 8 * h) * 2], ol = spare_ml[(wr * 16 + g + 8 * h) * 2 + 1];
              const float over = fmaxf(m[h], om), base = over == -INFINITY ? 0.f : over;
              mine[h] = fast_exp2(m[h] - base), other[h] = fast_exp2(om - base);
              l[h] = l[h] * mine[h] + ol * other[h];
              m[h] = over;
            }
#pragma unroll
            for (int n = 0; n < HALF; ++n)
              if (n0 + n < NT_O) {
                const float2 v = *reinterpret_cast<const float2*>(from + 8 * n + 2 * t4);
                o[n0 + n][2 * h] = o[n0 + n][2 * h] * mine[h] + (other[h] != 0.f ? v.x * other[h] : 0.f);
                o[n0 + n][2 * h + 1] = o[n0 + n][2 * h + 1] * mine[h] + (other[h] != 0.f ? v.y * other[h] : 0.f);
              }
          }
        }
        __syncthreads();
      }
    }
    if (wk == 0) {
      // The whole item is this block's where it begins and ends here.
      const bool whole = !(first && halfway) && now.tile + 1 == now.tiles;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (!whole) {
          const size_t slot = 2 * (size_t)blockIdx.x + (first ? 0 : 1), row = slot * ROWS + 16 * wr + g + 8 * h;
          if (t4 == 0) a.part_ml[2 * row] = m[h], a.part_ml[2 * row + 1] = l[h];
#pragma unroll
          for (int n = 0; n < NT_O; ++n)
            if (8 * n < D) *reinterpret_cast<float2*>(a.part_o + row * D + 8 * n + 2 * t4) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
          continue;
        }
        if (node[h] < 0) continue;
        const int token = now.k.first + node[h], head = now.head * group + (row0 + g + 8 * h) % group;
        float over = l[h], f = 1.f;
        if (a.sink) {
          const float z = a.sink[head] * LOG2E, base = fmaxf(m[h], z);
          f = fast_exp2(m[h] - base), over = l[h] * f + fast_exp2(z - base);
        }
        const float by = over > 0.f || over != over ? f / over : 0.f;
        bf16* out = static_cast<bf16*>(a.out) + (size_t)token * a.nq * D + head * D;
        const bf16* gate = a.gate ? static_cast<const bf16*>(a.gate) + (size_t)token * a.gate_stride + head * D : nullptr;
#pragma unroll
        for (int n = 0; n < NT_O; ++n)
          if (8 * n < D) {
            float y0 = o[n][2 * h] * by, y1 = o[n][2 * h + 1] * by;
            if (by == 0.f) y0 = y1 = 0.f;
            if (gate) {
              y0 *= tree_sigmoid(__bfloat162float(gate[8 * n + 2 * t4]));
              y1 *= tree_sigmoid(__bfloat162float(gate[8 * n + 2 * t4 + 1]));
            }
            *reinterpret_cast<unsigned*>(out + 8 * n + 2 * t4) = pack(y0, y1);
          }
      }
    }
    OMNIA_TRACE_BLOCK(6);  // its rows are out
    first = false, entered = true;
    now.next(a, shares);
  }
}

namespace {

template <int WR>
int launch(const TreeAttention& a, int blocks, cudaStream_t stream) {
  constexpr int HALF = NT_O > 8 ? (NT_O + 1) / 2 : NT_O;
  constexpr int bytes = STAGES * STAGE * 2 + (WR < WARPS ? WR * 16 * (8 * HALF + 4 + 2) * 4 : 0);
  static bool ready[64] = {};
  int device = 0;
  cudaGetDevice(&device);
  if (device < 0 || device >= 64) return (int)cudaErrorInvalidDevice;
  if (!ready[device]) {
    const cudaError_t e = cudaFuncSetAttribute(tree_shares_kernel<WR>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return (int)e;
    ready[device] = true;
  }
  launch_pdl(tree_shares_kernel<WR>, dim3(blocks), dim3(THREADS), bytes, stream, a);
  return OMNIA_LAUNCH_RESULT();
}

}  // namespace

// `rows`: of a tile, 16, 32 or 64; `blocks`: what the work is shared out over, with two slots of rows each in part_o and part_ml.
extern "C" int omnia_tree_attention_tc(const TreeAttention* given, int most_nodes, int rows, int blocks, void* stream) {
  TreeAttention a = *given;
  if (a.d != D || a.dv != D || a.requests < 1 || a.requests > TREE_MOST_REQUESTS || a.nkv < 1 || a.nkv > 65535 || a.nq % a.nkv || blocks < 1 ||
      most_nodes < 1 || (rows != 16 && rows != 32 && rows != 64))
    return (int)cudaErrorInvalidValue;
  a.parts = tree_row_tiles(a, most_nodes, rows);
  const cudaStream_t s = (cudaStream_t)stream;
  int code;
  if (rows == 16) code = launch<1>(a, blocks, s);
  else if (rows == 32) code = launch<2>(a, blocks, s);
#if HEAD_DIM <= 128
  else if (rows == 64) code = launch<4>(a, blocks, s);
#endif
  else return (int)cudaErrorInvalidValue;
  if (code) return code;
  return tree_join<bf16, D>(a, {rows, KEYS, 1, EXTRA}, most_nodes, blocks, s);
}
