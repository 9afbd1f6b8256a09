// What a caller's options do to float32 logits ahead of the choice of a token: penalties for tokens that have occurred, biases, and a
// mask of the tokens that a grammar allows. For a row's token v with logit z:
//   repetition p:  z > 0 ? z / p : z p          where v occurs in the row's text (or in the last `context` tokens of it)
//   frequency f, presence g:  z - f n - g       where v occurs n > 0 times in what was generated
//   bias:          z + the sum of the row's biases of v
//   mask:          -infinity where the row's mask has no bit for v
// The text is the request's history, prompt and generated tokens, and for a row of a drafted tree the drafted tokens on its way.
//
// A block has a slice of SLICE tokens of a row. It asks for its logits, and while they come counts the occurrences of its own tokens in shared
// memory: it reads the whole history (kilobytes, out of L2) and, of a drafted tree, the row's way, and keeps the entries of the biases' list that are
// its own, in their order. So there are no counts in device memory to hold, clear or share, integers are all that is added without an order,
// and no block waits for another. A slice is 8,192 tokens: an SM holds five such blocks, and a
// text is read by 19 of them where the vocabulary is 151,936. (Clusters whose blocks read a part of the history each and add to one another's counts: 64 rows of 24,000 tokens
// 48 us in place of 53, but 21 in place of 14 where the history is short.) What bounds a new tensor of many rows is memory, 8 bytes a logit: 512
// rows of 151,936 under masks, with texts of 2,000 tokens, 631 MB in 121 us (5.2 TB/s, 79 % of a copy's rate); 64 rows with texts of 6,000 and 40 biases
// take 20.6 us of a replayed graph and 25.7 with cold caches, 12.0 of them memory, the rest the texts in all of a row's blocks; a row alone 5.0. In place only what changes is touched.
// All is float32; what is counted are integers, so the order of additions to shared memory changes nothing.
#include "common.cuh"

struct AdjustLogits {
  const float* logits;
  float* out;
  const int* requests;                      // [rows] or null: row i is request i
  const int* history;                       // tokens of all requests
  const long long* starts;                  // [requests]
  const int *lengths, *prompts, *contexts;  // [requests]; contexts: or null
  const float *repetition, *frequency, *presence;  // [requests] or null
  const int* bias_ids;
  const float* bias_values;
  const int* bias_starts;                   // [requests + 1] or null
  const int *mask_words, *mask_rows;        // [masks, mask_width], [rows] or null
  const int *ancestors, *token_ids, *cu_seqlens, *nodes;  // drafted rows: [tokens, words], [tokens], [requests + 1], [rows], or null
  int* err;
  long long stride, out_stride, history_tokens, bias_count;
  int rows, vocab, num_requests, masks, mask_width, words, tokens, unused, penalised;
};

namespace {

constexpr int THREADS = 256, SLICE = 8192, LIST = 1024;  // entries of a list of biases that shared memory has room for
constexpr int EACH = SLICE / THREADS;       // logits of a thread
constexpr unsigned BIASED = 0x40000000u;    // of a count: the token has an entry in the list of biases
constexpr unsigned SEEN = 0x80000000u;      // of a count: the repetition penalty sees the token (all that is counted, where there is no context)

struct Penalties {
  float repetition, frequency, presence;
  unsigned seen;  // the bits of a count that the repetition penalty goes by
};
__device__ __forceinline__ float adjusted(float z, unsigned count, const Penalties& p) {
  if (count & p.seen & ~BIASED) z = z > 0.f ? z / p.repetition : z * p.repetition;
  const unsigned times = count & ~(SEEN | BIASED);
  if (times) z = z - p.frequency * (float)times - p.presence;
  return z;
}

// Additions to shared memory without a branch: nearly all of a text's tokens are other blocks', and a branch that a lane in a warp takes costs all.
__device__ __forceinline__ void add_if_below(unsigned* counts, unsigned at, unsigned end) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.lt.u32 p, %1, %2;\n\t@p red.shared::cta.add.u32 [%0], 1;\n\t}"
               ::"r"((unsigned)__cvta_generic_to_shared(counts) + 4 * at), "r"(at), "r"(end)
               : "memory");
}
__device__ __forceinline__ void or_if_below(unsigned* counts, unsigned at, unsigned end) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.lt.u32 p, %1, %2;\n\t@p red.shared::cta.or.b32 [%0], %3;\n\t}"
               ::"r"((unsigned)__cvta_generic_to_shared(counts) + 4 * at), "r"(at), "r"(end), "r"(SEEN)
               : "memory");
}
// The block's threads go through tokens [from, to): four at a time from the first 16-byte boundary on, what is ahead of it and behind the last one by one.
template <typename F>
__device__ __forceinline__ void scan(const int* tokens, int from, int to, F f) {
  const int* text = tokens + from;
  const int length = to - from, head = min(max(length, 0), (int)((16 - (reinterpret_cast<uintptr_t>(text) & 15)) & 15) / 4), quads = (length - head) / 4;
  const int tid = threadIdx.x;
  if (tid < head) f(text[tid]);
  if (tid < length - head - 4 * quads) f(text[head + 4 * quads + tid]);
  const int4* four = reinterpret_cast<const int4*>(text + head);
#pragma unroll 4
  for (int i = tid; i < quads; i += THREADS) {
    const int4 v = four[i];
    f(v.x), f(v.y), f(v.z), f(v.w);
  }
}

// IN_PLACE: only logits that change are read or written. VEC: logits of a 16-byte access.
template <bool IN_PLACE, int VEC>
__global__ void __launch_bounds__(THREADS, 5) adjust_logits_kernel(const __grid_constant__ AdjustLogits a) {
  __shared__ __align__(16) unsigned counts[SLICE];
  __shared__ int2 list[LIST];  // of the slice's biases: token, value
  __shared__ int listed[THREADS / 32];
  __shared__ unsigned allowed[SLICE / 32];  // the mask's bits for the slice
  static_assert(SLICE / 32 == THREADS, "a word of the mask a thread");
  pdl_wait();
  pdl_launch_dependents();
  const int lo = blockIdx.x * SLICE, hi = min(lo + SLICE, a.vocab), row = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const float* in = a.logits + row * a.stride;
  float* out = a.out + row * a.out_stride;
  // The logits come as far as L2 while the tokens are counted (kept in registers they cost an SM its fifth block).
  if constexpr (!IN_PLACE)
    if (lo + tid * 32 < hi) asm volatile("prefetch.global.L2 [%0];" ::"l"(in + lo + tid * 32));
  int request = a.requests ? a.requests[row] : row;
  const int node = a.nodes ? a.nodes[row] : 0, mask = a.mask_rows ? a.mask_rows[row] : -1;
  constexpr int CHUNK = VEC == 4 ? 16 : 8;
  float z[CHUNK];
  auto fetch = [&](int c0) {
#pragma unroll
    for (int i = 0; i < CHUNK / VEC; ++i) {
      const int v = lo + c0 * THREADS + (i * THREADS + tid) * VEC;
      if constexpr (VEC == 4) {
        if (v < hi) *reinterpret_cast<float4*>(z + 4 * i) = __ldcs(reinterpret_cast<const float4*>(in + v));
      } else {
        if (v < hi) z[i] = __ldcs(in + v);
      }
    }
  };
  const bool masked = mask >= 0 && mask < a.masks;
  if (mask >= a.masks && tid == 0) atomicOr(a.err, OMNIA_ERR_WORK);
  if (masked) allowed[tid] = lo / 32 + tid < a.mask_width ? (unsigned)a.mask_words[(size_t)mask * a.mask_width + lo / 32 + tid] : 0u;
  if (request < 0 || request >= a.num_requests) {
    if (tid == 0) atomicOr(a.err, OMNIA_ERR_WORK);
    request = -1;
  }
  int begin = 0, end = 0;
  if (a.bias_starts && request >= 0) {
    begin = a.bias_starts[request], end = a.bias_starts[request + 1];
    if (begin < 0 || end < begin || end > a.bias_count) {
      if (tid == 0) atomicOr(a.err, OMNIA_ERR_WORK);
      begin = end = 0;
    }
  }
  const bool counting = a.penalised && request >= 0, short_list = end > begin && end - begin <= LIST;
  Penalties p = {1.f, 0.f, 0.f, a.contexts ? SEEN : ~0u};
  int entries = 0;
  if (counting || short_list) {
    long long start = 0;
    int length = 0, prompt = 0, first = 0, drafted = 0, sight = 0;
    const unsigned* way = nullptr;
    if (counting) {
      start = a.starts[request], length = a.lengths[request], prompt = a.prompts[request];
      if (a.repetition) p.repetition = a.repetition[request];
      if (a.frequency) p.frequency = a.frequency[request];
      if (a.presence) p.presence = a.presence[request];
      if (start < 0 || length < 0 || start > a.history_tokens - length) {
        if (tid == 0) atomicOr(a.err, OMNIA_ERR_WORK);
        length = 0;
      }
      if (a.nodes) {
        first = a.cu_seqlens[request];
        if (node < first || node >= a.tokens || node - first >= 32 * a.words || first < 0) {
          if (tid == 0) atomicOr(a.err, OMNIA_ERR_WORK);
        } else {
          way = reinterpret_cast<const unsigned*>(a.ancestors) + (size_t)node * a.words;
        }
      }
      // The first token of the text that the repetition penalty sees.
      const int context = a.contexts ? a.contexts[request] : 0;
      if (context > 0) {
        if (way)
          for (int w = 0; w < a.words; ++w) drafted += __popc(way[w]);
        sight = max(length + drafted - context, 0);
      }
    }
    // A thread has four biases that follow one another.
    constexpr int PER = LIST / THREADS;
    static_assert(PER == 4, "four entries a thread");
    int ids[PER], mine = 0;
    float values[PER];
    if (short_list) {
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int e = begin + PER * tid + k, v = e < end ? a.bias_ids[e] : -1;
        values[k] = e < end ? a.bias_values[e] : 0.f;
        if (e < end && (v < 0 || v >= a.vocab)) atomicOr(a.err, OMNIA_ERR_TOKEN_ID);
        ids[k] = v >= lo && v < hi ? v : -1;
      }
    }
#pragma unroll
    for (int i = 0; i < SLICE / 4 / THREADS; ++i) reinterpret_cast<uint4*>(counts)[i * THREADS + tid] = make_uint4(0u, 0u, 0u, 0u);
    __syncthreads();
    if (counting) {
      // What is generated is counted; of the rest it matters that it is in the repetition penalty's sight (without a context whatever is counted is).
      const int* text = a.history + start;
      const int made = min(max(prompt, 0), length), seen0 = a.contexts ? min(max(sight, 0), length) : 0, seen1 = a.contexts ? length : made;
      scan(text, made, length, [&](int v) { add_if_below(&counts[0], (unsigned)(v - lo), (unsigned)(hi - lo)); });
      scan(text, seen0, seen1, [&](int v) { or_if_below(&counts[0], (unsigned)(v - lo), (unsigned)(hi - lo)); });
      if (blockIdx.x == 0)
        scan(text, 0, length, [&](int v) {
          if ((unsigned)v >= (unsigned)a.vocab) atomicOr(a.err, OMNIA_ERR_TOKEN_ID);
        });
      if (way) {
        for (int j = tid; j < 32 * a.words; j += THREADS)
          if ((way[j >> 5] >> (j & 31)) & 1u) {
            int at = length;  // its place in the text: behind the history and what is above it on the way
            for (int w = 0; w <= j >> 5; ++w) at += __popc(w < j >> 5 ? way[w] : way[w] & ((1u << (j & 31)) - 1u));
            const int v = first + j < a.tokens ? a.token_ids[first + j] : -1;
            if (v >= lo && v < hi) {
              atomicAdd(&counts[v - lo], 1u);
              if (a.contexts && at >= sight) atomicOr(&counts[v - lo], SEEN);
            } else if ((unsigned)v >= (unsigned)a.vocab && blockIdx.x == 0) {
              atomicOr(a.err, OMNIA_ERR_TOKEN_ID);
            }
          }
      }
    }
    if (short_list) {
      // The slice's entries in the list's order.
#pragma unroll
      for (int k = 0; k < PER; ++k) mine += ids[k] >= 0;
      int upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const int other = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += other;
      }
      if (lane == 31) listed[warp] = upto;
      __syncthreads();
      int at = upto - mine;
#pragma unroll
      for (int w = 0; w < THREADS / 32; ++w) {
        if (w < warp) at += listed[w];
        entries += listed[w];
      }
#pragma unroll
      for (int k = 0; k < PER; ++k)
        if (ids[k] >= 0) {
          list[at++] = make_int2(ids[k], __float_as_int(values[k]));
          atomicOr(&counts[ids[k] - lo], BIASED);
        }
    }
  }
  if constexpr (!IN_PLACE) fetch(0);
  __syncthreads();
  const bool changing = counting || entries > 0;
  auto changed = [&](float y, int v, unsigned count) {
    y = adjusted(y, count, p);
    if (count & BIASED)
#pragma unroll 1
      for (int e = 0; e < entries; ++e)
        if (list[e].x == v) y += __int_as_float(list[e].y);
    return y;
  };
  if (!IN_PLACE || masked || changing) {
#pragma unroll 1
    for (int c0 = 0; c0 < EACH; c0 += CHUNK) {
      if constexpr (!IN_PLACE)
        if (c0) fetch(c0);
#pragma unroll
      for (int i = 0; i < CHUNK / VEC; ++i) {
        const int v = lo + c0 * THREADS + (i * THREADS + tid) * VEC;
        if (v >= hi) continue;
        const unsigned bits = masked ? allowed[(v - lo) >> 5] >> (v & 31) : ~0u;
        unsigned count[VEC] = {}, any = 0;
        if (changing) {
          if constexpr (VEC == 4) {
            *reinterpret_cast<uint4*>(count) = *reinterpret_cast<const uint4*>(counts + (v - lo));
            any = count[0] | count[1] | count[2] | count[3];
          } else {
            any = count[0] = counts[v - lo];
          }
        }
        if constexpr (IN_PLACE) {
#pragma unroll
          for (int k = 0; k < VEC; ++k) {
            if (!((bits >> k) & 1u)) out[v + k] = -INFINITY;
            else if (count[k]) out[v + k] = changed(in[v + k], v + k, count[k]);
          }
        } else {
          if (any) {
#pragma unroll
            for (int k = 0; k < VEC; ++k)
              if (count[k]) z[VEC * i + k] = changed(z[VEC * i + k], v + k, count[k]);
          }
          float y[VEC];
#pragma unroll
          for (int k = 0; k < VEC; ++k) y[k] = (bits >> k) & 1u ? z[VEC * i + k] : -INFINITY;
          if constexpr (VEC == 4) __stcs(reinterpret_cast<float4*>(out + v), *reinterpret_cast<float4*>(y));
          else __stcs(out + v, y[0]);
        }
      }
    }
  }
  if (end - begin > LIST) {
    // A long list: a warp has an eighth of the slice and reads all entries, 32 at a time: so a token's are added in their order.
    __syncthreads();
    const int from = lo + warp * (SLICE / (THREADS / 32)), to = min(from + SLICE / (THREADS / 32), hi);
    for (int e0 = begin; e0 < end; e0 += 32) {
      const int v = e0 + lane < end ? a.bias_ids[e0 + lane] : -1;
      if (e0 + lane < end && (v < 0 || v >= a.vocab)) atomicOr(a.err, OMNIA_ERR_TOKEN_ID);
      const bool mine = v >= from && v < to;
      if (!__any_sync(0xffffffffu, mine)) continue;
      const float value = mine ? a.bias_values[e0 + lane] : 0.f;
      const unsigned same = __match_any_sync(0xffffffffu, mine ? v : -1 - lane);
      float y = 0.f;
      if (mine) y = out[v];
      // Every lane of a token adds the token's entries in their order; the first writes.
      for (int k = 0; k < 32; ++k) {
        const float other = __shfl_sync(0xffffffffu, value, k);
        if ((same >> k) & 1u) y += other;
      }
      if (mine && (same & ((1u << lane) - 1u)) == 0 && out[v] != -INFINITY) out[v] = y;
      __syncwarp();
    }
  }
}

}  // namespace

extern "C" int omnia_adjust_logits(const AdjustLogits* given, int in_place, void* stream) {
  AdjustLogits a = *given;
  if (a.rows < 1 || a.vocab < 1) return a.rows < 0 || a.vocab < 1 ? (int)cudaErrorInvalidValue : 0;
  const int slices = (a.vocab + SLICE - 1) / SLICE;
  if (a.rows > 65535) return (int)cudaErrorInvalidValue;
  const bool vec = ((uintptr_t)a.logits | (uintptr_t)a.out) % 16 == 0 && a.stride % 4 == 0 && a.out_stride % 4 == 0 && a.vocab % 4 == 0;
  const dim3 grid(slices, a.rows);
  const cudaStream_t s = (cudaStream_t)stream;
  if (in_place) launch_pdl(vec ? adjust_logits_kernel<true, 4> : adjust_logits_kernel<true, 1>, grid, dim3(THREADS), 0, s, a);
  else launch_pdl(vec ? adjust_logits_kernel<false, 4> : adjust_logits_kernel<false, 1>, grid, dim3(THREADS), 0, s, a);
  return OMNIA_LAUNCH_RESULT();
}
