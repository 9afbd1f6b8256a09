// What a caller's options do to float32 logits ahead of the choice of a token: penalties for tokens that have occurred, biases, and a
// mask of the tokens that a grammar allows. For a row's token v with logit z:
//   repetition p:  z > 0 ? z / p : z p          where v occurs in the row's text (or in the last `context` tokens of it)
//   frequency f, presence g:  z - f n - g       where v occurs n > 0 times in what was generated
//   bias:          z + the sum of the row's biases of v
//   mask:          -infinity where the row's mask has no bit for v
// The text is the request's history, prompt and generated tokens, and for a row of a drafted tree the drafted tokens on its way.
//
// A block has a slice of SLICE tokens of some rows that come one after the other. It counts the occurrences of its own tokens in shared
// memory: it reads the whole history (kilobytes, out of L2, once for the rows of one request), and adds a row's drafted tokens for that row alone.
// So there are no counts in device memory to hold, clear or share, integers are all that is added without an order, and no block waits
// for another. What bounds a new tensor of many rows is memory, 8 bytes a logit; in place only what changes is touched.
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
  int rows, vocab, num_requests, masks, mask_width, words, tokens, each, penalised;  // each: rows of a block
};

namespace {

constexpr int THREADS = 256, SLICE = 8192;
constexpr int EACH = SLICE / THREADS;       // logits of a thread
constexpr unsigned SEEN = 0x80000000u;      // of a count: the repetition penalty sees the token (all that is counted, where there is no context)

struct Penalties {
  float repetition, frequency, presence;
  unsigned seen;  // the bits of a count that the repetition penalty goes by
};
__device__ __forceinline__ float adjusted(float z, unsigned count, const Penalties& p) {
  if (count & p.seen) z = z > 0.f ? z / p.repetition : z * p.repetition;
  const unsigned times = count & ~SEEN;
  if (times) z = z - p.frequency * (float)times - p.presence;
  return z;
}

// IN_PLACE: only logits that change are read or written. VEC: logits of a 16-byte access.
template <bool IN_PLACE, int VEC>
__global__ void __launch_bounds__(THREADS) adjust_logits_kernel(const __grid_constant__ AdjustLogits a) {
  __shared__ __align__(16) unsigned counts[SLICE];
  pdl_wait();
  pdl_launch_dependents();
  const int lo = blockIdx.x * SLICE, hi = min(lo + SLICE, a.vocab);
  const bool penalised = a.penalised;
  int counted = -1;  // the request whose history the counts are of
  const int row0 = blockIdx.y * a.each, row1 = min(row0 + a.each, a.rows);
  for (int row = row0; row < row1; ++row) {
    int request = a.requests ? a.requests[row] : row;
    if (request < 0 || request >= a.num_requests) {
      if (threadIdx.x == 0) atomicOr(a.err, OMNIA_ERR_WORK);
      request = -1;
    }
    const float* in = a.logits + row * a.stride;
    float* out = a.out + row * a.out_stride;
    // The row's logits (the first of them, one by one) are on their way while its tokens are counted.
    constexpr int CHUNK = VEC == 4 ? EACH : 8;
    float z[CHUNK];
    auto fetch = [&](int c0) {
#pragma unroll
      for (int i = 0; i < CHUNK / VEC; ++i) {
        const int v = lo + c0 * THREADS + (i * THREADS + threadIdx.x) * VEC;
        if constexpr (VEC == 4) {
          if (v < hi) *reinterpret_cast<float4*>(z + 4 * i) = __ldcs(reinterpret_cast<const float4*>(in + v));
        } else {
          if (v < hi) z[i] = __ldcs(in + v);
        }
      }
    };
    if constexpr (!IN_PLACE) fetch(0);
    Penalties p = {1.f, 0.f, 0.f, a.contexts ? SEEN : ~0u};
    const bool counting = penalised && request >= 0;
    int length = 0, prompt = 0, drafted = 0, sight = 0, first = 0;
    long long start = 0;
    const unsigned* way = nullptr;
    if (counting) {
      if (a.repetition) p.repetition = a.repetition[request];
      if (a.frequency) p.frequency = a.frequency[request];
      if (a.presence) p.presence = a.presence[request];
      start = a.starts[request], length = a.lengths[request], prompt = a.prompts[request];
      if (start < 0 || length < 0 || start + length > a.history_tokens) {
        if (threadIdx.x == 0) atomicOr(a.err, OMNIA_ERR_WORK);
        length = 0;
      }
      if (a.nodes) {
        const int node = a.nodes[row];
        first = a.cu_seqlens[request];
        if (node < first || node >= a.tokens || node - first >= 32 * a.words || first < 0) {
          if (threadIdx.x == 0) atomicOr(a.err, OMNIA_ERR_WORK);
        } else {
          way = reinterpret_cast<const unsigned*>(a.ancestors) + (size_t)node * a.words;
          for (int w = 0; w < a.words; ++w) drafted += __popc(way[w]);
        }
      }
      // The first token of the text that the repetition penalty sees.
      const int context = a.contexts ? a.contexts[request] : 0;
      sight = context > 0 ? max(length + drafted - context, 0) : 0;
    }
    // A context's beginning moves with the row's drafted tokens, so such rows are counted one by one.
    if (counting && (request != counted || (a.contexts && a.nodes))) {
      __syncthreads();
      for (int i = threadIdx.x; i < SLICE / 4; i += THREADS) reinterpret_cast<uint4*>(counts)[i] = make_uint4(0u, 0u, 0u, 0u);
      __syncthreads();
      const int* text = a.history + start;
      for (int i = threadIdx.x; i < length; i += THREADS) {
        const int v = text[i];
        if (v >= lo && v < hi) {
          if (i >= prompt) atomicAdd(&counts[v - lo], 1u);
          if (i >= sight) atomicOr(&counts[v - lo], SEEN);
        } else if ((v < 0 || v >= a.vocab) && blockIdx.x == 0) {
          atomicOr(a.err, OMNIA_ERR_TOKEN_ID);
        }
      }
      counted = request;
    }
    if (way) {
      __syncthreads();
      for (int j = threadIdx.x; j < 32 * a.words; j += THREADS)
        if ((way[j >> 5] >> (j & 31)) & 1u) {
          const int v = first + j < a.tokens ? a.token_ids[first + j] : -1;
          if (v >= lo && v < hi) {
            atomicAdd(&counts[v - lo], 1u);
            if (a.contexts) {  // (its place in the text: behind the history and what is above it on the way)
              int above = length;
              for (int w = 0; w <= j >> 5; ++w) above += __popc(w < j >> 5 ? way[w] : way[w] & ((1u << (j & 31)) - 1u));
              if (above >= sight) atomicOr(&counts[v - lo], SEEN);
            }
          } else if ((v < 0 || v >= a.vocab) && blockIdx.x == 0) {
            atomicOr(a.err, OMNIA_ERR_TOKEN_ID);
          }
        }
    }
    if (counting) __syncthreads();
    const int mask = a.mask_rows ? a.mask_rows[row] : -1;
    const bool masked = mask >= 0 && mask < a.masks;
    if (mask >= a.masks && threadIdx.x == 0) atomicOr(a.err, OMNIA_ERR_WORK);
    const unsigned* allowed = masked ? reinterpret_cast<const unsigned*>(a.mask_words) + (size_t)mask * a.mask_width : nullptr;
#pragma unroll 1
    for (int c0 = 0; c0 < EACH; c0 += CHUNK) {
      if constexpr (!IN_PLACE)
        if (c0) fetch(c0);
#pragma unroll
      for (int i = 0; i < CHUNK / VEC; ++i) {
        const int v = lo + c0 * THREADS + (i * THREADS + threadIdx.x) * VEC;
        if (v >= hi) continue;
        const unsigned bits = masked ? allowed[v >> 5] >> (v & 31) : ~0u;
        unsigned count[VEC];
        if constexpr (VEC == 4) {
          *reinterpret_cast<uint4*>(count) = counting ? *reinterpret_cast<const uint4*>(counts + (v - lo)) : make_uint4(0u, 0u, 0u, 0u);
        } else {
          count[0] = counting ? counts[v - lo] : 0u;
        }
        if constexpr (IN_PLACE) {
#pragma unroll
          for (int k = 0; k < VEC; ++k) {
            if (!((bits >> k) & 1u)) out[v + k] = -INFINITY;
            else if (count[k]) out[v + k] = adjusted(in[v + k], count[k], p);
          }
        } else {
          float y[VEC];
#pragma unroll
          for (int k = 0; k < VEC; ++k)
            y[k] = !((bits >> k) & 1u) ? -INFINITY : count[k] ? adjusted(z[VEC * i + k], count[k], p) : z[VEC * i + k];
          if constexpr (VEC == 4) *reinterpret_cast<float4*>(out + v) = *reinterpret_cast<float4*>(y);
          else out[v] = y[0];
        }
      }
    }
    if (way) {
      __syncthreads();
      for (int j = threadIdx.x; j < 32 * a.words; j += THREADS)
        if ((way[j >> 5] >> (j & 31)) & 1u) {
          const int v = first + j < a.tokens ? a.token_ids[first + j] : -1;
          if (v >= lo && v < hi) atomicSub(&counts[v - lo], 1u);
        }
    }
    if (a.bias_starts && request >= 0) {
      // A warp has an eighth of the slice and reads the whole list, 32 entries at a time: so a token's entries are added in their order.
      __syncthreads();
      const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
      const int from = lo + warp * (SLICE / (THREADS / 32)), to = min(from + SLICE / (THREADS / 32), hi);
      int begin = a.bias_starts[request], end = a.bias_starts[request + 1];
      if (begin < 0 || end < begin || end > a.bias_count) {
        if (threadIdx.x == 0) atomicOr(a.err, OMNIA_ERR_WORK);
        begin = end = 0;
      }
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
}

}  // namespace

extern "C" int omnia_adjust_logits(const AdjustLogits* given, int in_place, void* stream) {
  AdjustLogits a = *given;
  if (a.rows < 1 || a.vocab < 1) return a.rows < 0 || a.vocab < 1 ? (int)cudaErrorInvalidValue : 0;
  const int slices = (a.vocab + SLICE - 1) / SLICE;
  a.each = a.nodes ? 8 : 1;  // neighbours in a tree have one history
  const long long blocks = (a.rows + a.each - 1) / a.each;
  if (blocks > 65535) return (int)cudaErrorInvalidValue;
  const bool vec = ((uintptr_t)a.logits | (uintptr_t)a.out) % 16 == 0 && a.stride % 4 == 0 && a.out_stride % 4 == 0 && a.vocab % 4 == 0;
  const dim3 grid(slices, (unsigned)blocks);
  const cudaStream_t s = (cudaStream_t)stream;
  if (in_place) launch_pdl(vec ? adjust_logits_kernel<true, 4> : adjust_logits_kernel<true, 1>, grid, dim3(THREADS), 0, s, a);
  else launch_pdl(vec ? adjust_logits_kernel<false, 4> : adjust_logits_kernel<false, 1>, grid, dim3(THREADS), 0, s, a);
  return OMNIA_LAUNCH_RESULT();
}
