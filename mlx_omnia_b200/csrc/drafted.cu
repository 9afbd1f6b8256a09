// What a step that reads drafted tokens needs around its layers: its tables, made on the GPU from the requests' lengths and lists of
// pages; the path of drafts that the model agrees with; and the kept tokens' rows of the cache, moved to where a request that had brought
// only these would have them.
//
// A request's drafted tokens (its nodes) are numbered 0, 1, ... in the order they are brought; node 0 is known, each other one goes on from
// an earlier one, its parent. What a node descends from, itself too, is a row of bits (its ancestors), `words` words of 32 bits.
#include <stddef.h>
#include <string.h>

#include "common.cuh"

namespace {

constexpr int THREADS = 256;
constexpr int MOST_WORDS = 8, MOST_NODES = 32 * MOST_WORDS;  // a node a thread
constexpr int MOST_GROUPS = 8, MOST_KINDS = 8;
static_assert(MOST_NODES == THREADS, "a node a thread");

}  // namespace

// One group of caches: where each request's list of pages begins, and the table and the slots that are made from them.
struct TableGroup {
  const int* pages;
  const long long* starts;  // [requests]
  int* table;               // [requests, width]
  long long* slots;         // [tokens]
  long long count;          // of `pages`
  int width, stride;
};
struct StepTables {
  const int *held, *brought, *parents;  // [requests], [requests], [tokens] or null
  int *positions, *cu_seqlens, *seq_lens, *ancestors, *err;
  int requests, tokens, page_size, words, groups;
  TableGroup group[MOST_GROUPS];
};

namespace {

// The sum of `brought` ahead of request `upto` (a request that says less than nothing brings nothing).
__device__ long long tokens_ahead(const int* brought, int upto, long long* sums) {
  long long mine = 0;
  for (int i = threadIdx.x; i < upto; i += THREADS) mine += max(brought[i], 0);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = mine;
  __syncthreads();
  long long all = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) all += sums[w];
  return all;
}

// Bytes: 8 a token and table (its slot), 4 a column, 8 and the bits of its ancestors a token: 1.8 MB for 64 requests of 32,768 positions with 64 tokens in two
// groups of caches, 0.3 us of memory; what it takes, 5.8 us of a replayed graph (8 requests with a token: 2.6), is a launch, a few dependent
// reads of L2 (what is brought, where a list begins, the list) and, of trees, a round through shared memory for every doubling of a request's tokens.
//
// A block's row of the grid is a request (the last row: the tokens behind the last request's); the blocks of a row share its tokens and its
// tables' columns. Each adds up for itself how many tokens come ahead: a few kilobytes out of L2, in place of a launch of its own.
__global__ void __launch_bounds__(THREADS) step_tables_kernel(const __grid_constant__ StepTables a) {
  __shared__ long long sums[THREADS / 32];
  __shared__ unsigned bits[MOST_NODES][MOST_WORDS];
  __shared__ int up[MOST_NODES];
  pdl_wait();
  pdl_launch_dependents();
  const int r = blockIdx.y, part = blockIdx.x, parts = gridDim.x;
  const long long ahead = tokens_ahead(a.brought, r, sums);
  const int first = (int)min(ahead, (long long)a.tokens);
  if (r == a.requests) {
    if (part == 0 && threadIdx.x == 0) {
      a.cu_seqlens[r] = first;
      if (ahead > a.tokens) atomicOr(a.err, OMNIA_ERR_WORK);
    }
    for (int t = first + part * THREADS + threadIdx.x; t < a.tokens; t += parts * THREADS) {
      a.positions[t] = -1;
      for (int g = 0; g < a.groups; ++g) a.group[g].slots[t] = -1;
      if (a.ancestors)
        for (int w = 0; w < a.words; ++w) a.ancestors[(size_t)t * a.words + w] = 0;
    }
    return;
  }
  const int held = a.held[r], wanted = max(a.brought[r], 0);
  int count = min(wanted, a.tokens - first);
  const bool beyond = (long long)held + count > 0x7fffffffLL;  // positions are numbers of 31 bits
  const bool padding = held < 0 || beyond;                     // a request that is there for the step's shape only
  if (part == 0 && threadIdx.x == 0) {
    if (beyond) atomicOr(a.err, OMNIA_ERR_WORK);
    a.cu_seqlens[r] = first;
    a.seq_lens[r] = padding ? 0 : held + count;
  }
  for (int g = 0; g < a.groups; ++g) {
    const TableGroup& group = a.group[g];
    const long long start = group.starts[r];
    const int rows = padding ? 0 : (int)(((long long)held + count + group.stride - 1) / group.stride);
    const int pages = (int)(((long long)rows + a.page_size - 1) / a.page_size);
    const bool fits = pages <= group.width && start >= 0 && start <= group.count - pages;
    if (!fits && pages && part == 0 && threadIdx.x == 0) atomicOr(a.err, OMNIA_ERR_WORK);
    int* table = group.table + (size_t)r * group.width;
    for (int c = part * THREADS + threadIdx.x; c < group.width; c += parts * THREADS)
      table[c] = fits && c < pages ? group.pages[start + c] : -1;
    for (int j = part * THREADS + threadIdx.x; j < count; j += parts * THREADS) {
      long long slot = -1;
      if (!padding && fits) {
        const int row = (held + j) / group.stride, page = group.pages[start + row / a.page_size];
        if (page >= 0) slot = (long long)page * a.page_size + row % a.page_size;
        else atomicOr(a.err, OMNIA_ERR_PAGE);
      }
      group.slots[first + j] = slot;
    }
  }
  if (!a.ancestors) {
    for (int j = part * THREADS + threadIdx.x; j < count; j += parts * THREADS) a.positions[first + j] = padding ? -1 : held + j;
    return;
  }
  if (part > 0) return;
  // A node's ancestors by doubling: what it knows of itself and its way up, joined with what the node at that way's end knows.
  if (count > 32 * a.words) {
    if (threadIdx.x == 0) atomicOr(a.err, OMNIA_ERR_WORK);
    for (int t = 32 * a.words + threadIdx.x; t < count; t += THREADS) {
      a.positions[first + t] = -1;
      for (int w = 0; w < a.words; ++w) a.ancestors[(size_t)(first + t) * a.words + w] = 0;
    }
    count = 32 * a.words;
  }
  const int j = threadIdx.x;
  unsigned mine[MOST_WORDS];
  int way = -1;
  if (j < count) {
    way = a.parents ? a.parents[first + j] : j - 1;
    if (way < -1 || way >= j) atomicOr(a.err, OMNIA_ERR_WORK), way = -1;
  }
#pragma unroll
  for (int w = 0; w < MOST_WORDS; ++w) mine[w] = j < count && j >> 5 == w ? 1u << (j & 31) : 0u;
  for (int span = 1; span < count; span *= 2) {
#pragma unroll
    for (int w = 0; w < MOST_WORDS; ++w) bits[j][w] = mine[w];
    up[j] = way;
    __syncthreads();
    if (way >= 0) {
#pragma unroll
      for (int w = 0; w < MOST_WORDS; ++w) mine[w] |= bits[way][w];
      way = up[way];
    }
    __syncthreads();
  }
  if (j < count) {
    int depth = -1;
#pragma unroll
    for (int w = 0; w < MOST_WORDS; ++w) {
      depth += __popc(mine[w]);
      if (w < a.words) a.ancestors[(size_t)(first + j) * a.words + w] = (int)(padding ? 0u : mine[w]);
    }
    a.positions[first + j] = padding ? -1 : held + depth;
  }
}

// A node is kept when every node on its way from node 0 is what was chosen behind its parent, the earliest of equal siblings. One
// node at most of each depth is, so the kept ones are the ancestors of the last of them. A block a request, a node a thread: a launch, two dependent reads
// and the siblings' comparison in shared memory (64 requests of 64: 2.4 us of a replayed graph, one of 12 2.1; what it reads and writes are some kilobytes).
__global__ void __launch_bounds__(THREADS)
accept_drafts_kernel(const int* chosen, const int* ids, const int* ancestors, const int* cu_seqlens, int words, int* path, int* kept,
                     int* tokens, int rows, int* err) {
  __shared__ int id[MOST_NODES], pick[MOST_NODES], parent[MOST_NODES];
  __shared__ unsigned right[MOST_WORDS], reached[MOST_WORDS];
  pdl_wait();
  pdl_launch_dependents();
  const int r = blockIdx.x, j = threadIdx.x, most = 32 * words, warp = j >> 5, lane = j & 31;
  const int first = cu_seqlens[r];
  int count = cu_seqlens[r + 1] - first;
  if (first < 0 || count < 0 || count > most || first + count > rows) {
    if (j == 0) atomicOr(err, OMNIA_ERR_WORK);
    count = first < 0 ? 0 : max(0, min(min(count, most), rows - first));
  }
  unsigned mine[MOST_WORDS];
  int up = -1;
#pragma unroll
  for (int w = 0; w < MOST_WORDS; ++w) {
    mine[w] = 0;
    if (j < count && w < words && w <= warp) {
      const unsigned all = (unsigned)ancestors[(size_t)(first + j) * words + w];
      const unsigned ahead = w < warp ? all : all & ((1u << lane) - 1u);
      if (ahead) up = 32 * w + 31 - __clz(ahead);
      mine[w] = w < warp ? ahead : ahead | (1u << lane);
    }
  }
  if (j < count) id[j] = ids[first + j], pick[j] = chosen[first + j];
  parent[j] = up;
  __syncthreads();
  bool good = j == 0;
  if (j > 0 && j < count && up >= 0 && id[j] == pick[up]) {
    good = true;
    for (int i = up + 1; i < j; ++i) good &= !(parent[i] == up && id[i] == id[j]);
  }
  const unsigned together = __ballot_sync(0xffffffffu, good && j < count);
  if (lane == 0) right[warp] = together;
  __syncthreads();
  bool reach = j < count;
#pragma unroll
  for (int w = 0; w < MOST_WORDS; ++w) reach &= (mine[w] & ~right[w]) == 0;
  const unsigned there = __ballot_sync(0xffffffffu, reach);
  if (lane == 0) reached[warp] = there;
  __syncthreads();
  int last = -1;
#pragma unroll
  for (int w = 0; w < MOST_WORDS; ++w)
    if (reached[w]) last = 32 * w + 31 - __clz(reached[w]);
  __syncthreads();
  if (j == last) {
#pragma unroll
    for (int w = 0; w < MOST_WORDS; ++w) right[w] = mine[w];
  }
  __syncthreads();
  int all = 0, ahead = 0;
  bool on = false;
  if (last >= 0) {
#pragma unroll
    for (int w = 0; w < MOST_WORDS; ++w) {
      all += __popc(right[w]);
      if (w < warp) ahead += __popc(right[w]);
      if (w == warp) ahead += __popc(right[w] & ((1u << lane) - 1u)), on = (right[w] >> lane) & 1u;
    }
  }
  if (on) path[(size_t)r * most + ahead] = j;
  if (j >= all && j < most) path[(size_t)r * most + j] = -1;
  if (j == 0) {
    kept[r] = all;
    tokens[r] = last >= 0 ? pick[last] : -1;
  }
}

struct KeepRows {
  char* pages;
  const int *table, *held, *path, *kept;
  int* err;
  long long layer_bytes, page_bytes;
  int requests, layers, num_pages, page_size, width, most, kinds, units;  // units: of U bytes, of a position's rows of all kinds
  int heads[MOST_KINDS], row_units[MOST_KINDS];                   // of each kind: heads, units of a head's row
};

// A block has one request's kept rows in some layers, a thread a unit of U bytes of a position's rows in turn: it reads four kept positions' in two
// layers and then writes them. A row goes to its own place or to an earlier one, and the rows of a path come in order, so what is written was
// read before, or belongs to a draft that is not kept. Bytes: 2 rows of all layers a kept token that moves. One request's 3 in 28 layers are 0.7 MB and take 3.0 us
// of a replayed graph, a launch and three dependent reads (which are kept, their pages, their rows); 64 requests' 76 in 36 layers 22 MB, 3.4 us at the memory's
// rate, 6.0 here (10.1 with a division by the page's size at every access in place of one a row).
template <typename U>
__global__ void __launch_bounds__(THREADS) keep_rows_kernel(const __grid_constant__ KeepRows a) {
  __shared__ long long from[MOST_NODES], to[MOST_NODES];  // where the page lies, in bytes from its layer's first one; -1: no move
  __shared__ int from_row[MOST_NODES], to_row[MOST_NODES], path[MOST_NODES], moves;
  pdl_wait();
  pdl_launch_dependents();
  const int r = blockIdx.x, j = threadIdx.x;
  const int held = a.held[r], count = held < 0 ? 0 : min(max(a.kept[r], 0), a.most);
  const int node = j < a.most ? a.path[(size_t)r * a.most + j] : -1;
  path[j] = node;
  if (j == 0) moves = 0;
  __syncthreads();
  const bool moved = j < count && node != j;
  if (moved) atomicAdd(&moves, 1);
  __syncthreads();
  if (moves == 0) return;
  // Nodes of a path only go up: once one has moved, all behind it have.
  const int skip = count - moves;
  if (j < count) {
    int source = -1, target = -1;
    if (moved && j >= skip && node > j && node < a.most && (j == 0 || node > path[j - 1])) {
      const long long sp = ((long long)held + node) / a.page_size, dp = ((long long)held + j) / a.page_size;
      if (sp < a.width) source = a.table[(size_t)r * a.width + sp], target = a.table[(size_t)r * a.width + dp];
    }
    const bool good = source >= 0 && target >= 0 && source < a.num_pages && target < a.num_pages;
    if (moved && !good && blockIdx.y == 0) atomicOr(a.err, OMNIA_ERR_PAGE);
    from[j] = good ? source * a.page_bytes : -1, from_row[j] = (int)(((long long)held + node) % a.page_size);
    to[j] = good ? target * a.page_bytes : -1, to_row[j] = (int)(((long long)held + j) % a.page_size);
  }
  __syncthreads();
  for (int unit = j; unit < a.units; unit += THREADS) {
    int rest = unit, kind = 0;
    long long base = 0;
    while (rest >= a.heads[kind] * a.row_units[kind]) {
      rest -= a.heads[kind] * a.row_units[kind];
      base += (long long)a.heads[kind] * a.row_units[kind] * a.page_size;
      ++kind;
    }
    const int width = a.row_units[kind], head = rest / width, column = rest % width;
    base += (long long)head * a.page_size * width + column;
    auto at = [&](int layer, long long page, int row) { return reinterpret_cast<U*>(a.pages + layer * a.layer_bytes + page) + base + (long long)row * width; };
    for (int l0 = blockIdx.y; l0 < a.layers; l0 += 2 * gridDim.y)
      for (int i0 = skip; i0 < count; i0 += 4) {
        U held_rows[2][4];
#pragma unroll
        for (int l = 0; l < 2; ++l)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (l0 + l * (int)gridDim.y < a.layers && i0 + i < count && from[i0 + i] >= 0) held_rows[l][i] = *at(l0 + l * gridDim.y, from[i0 + i], from_row[i0 + i]);
#pragma unroll
        for (int l = 0; l < 2; ++l)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (l0 + l * (int)gridDim.y < a.layers && i0 + i < count && from[i0 + i] >= 0) *at(l0 + l * gridDim.y, to[i0 + i], to_row[i0 + i]) = held_rows[l][i];
      }
  }
}

}  // namespace

// (What is given ends behind the last group.)
extern "C" int omnia_step_tables(const void* given, void* stream) {
  StepTables a = {};
  memcpy(&a, given, offsetof(StepTables, group));
  if (a.groups < 0 || a.groups > MOST_GROUPS || a.words < 0 || a.words > MOST_WORDS || a.requests < 1 || a.requests > 65534 || a.page_size < 1 ||
      a.tokens < 0)
    return (int)cudaErrorInvalidValue;
  memcpy(a.group, static_cast<const char*>(given) + offsetof(StepTables, group), a.groups * sizeof(TableGroup));
  int longest = a.tokens;
  for (int g = 0; g < a.groups; ++g) longest = max(longest, a.group[g].width);
  // Blocks enough for the widest table or the longest request, and no more than fill the GPU.
  const int wanted = (longest + 2 * THREADS - 1) / (2 * THREADS), room = 8 * omnia_sm_count() / (a.requests + 1);
  const int parts = max(1, min(wanted, room));
  launch_pdl(step_tables_kernel, dim3(parts, a.requests + 1), dim3(THREADS), 0, (cudaStream_t)stream, a);
  return OMNIA_LAUNCH_RESULT();
}

extern "C" int omnia_accept_drafts(const int* chosen, const int* ids, const int* ancestors, const int* cu_seqlens, int requests, int words,
                                   int* path, int* kept, int* tokens, int rows, int* err, void* stream) {
  if (words < 1 || words > MOST_WORDS || requests < 1) return (int)cudaErrorInvalidValue;
  launch_pdl(accept_drafts_kernel, dim3(requests), dim3(THREADS), 0, (cudaStream_t)stream, chosen, ids, ancestors, cu_seqlens, words, path, kept,
             tokens, rows, err);
  return OMNIA_LAUNCH_RESULT();
}

// `bytes`: of a head's row, by kind.
extern "C" int omnia_keep_rows(void* pages, long long layer_bytes, long long page_bytes, int layers, int num_pages, int page_size, const int* heads,
                               const int* bytes, int kinds, const int* table, int width, const int* held, const int* path, const int* kept,
                               int requests, int most, int* err, void* stream) {
  if (kinds < 1 || kinds > MOST_KINDS || requests < 1 || layers < 1 || layers > 65535 || most < 1 || most > MOST_NODES || page_size < 1 || width < 1)
    return (int)cudaErrorInvalidValue;
  KeepRows a = {};
  a.pages = (char*)pages, a.table = table, a.held = held, a.path = path, a.kept = kept, a.err = err;
  a.layer_bytes = layer_bytes, a.page_bytes = page_bytes;
  a.requests = requests, a.layers = layers, a.num_pages = num_pages, a.page_size = page_size, a.width = width, a.most = most, a.kinds = kinds;
  long long all = (long long)(uintptr_t)pages | layer_bytes | page_bytes;
  for (int k = 0; k < kinds; ++k) all |= bytes[k];
  const int unit = all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : all % 2 == 0 ? 2 : 1;
  for (int k = 0; k < kinds; ++k) a.heads[k] = heads[k], a.row_units[k] = bytes[k] / unit, a.units += heads[k] * a.row_units[k];
  // Blocks that the GPU holds at once, each with as many layers as that takes.
  const int room = 6 * omnia_sm_count() / requests;
  const dim3 grid(requests, room < 1 ? 1 : room < layers ? room : layers);
  const cudaStream_t s = (cudaStream_t)stream;
  if (unit == 16) launch_pdl(keep_rows_kernel<uint4>, grid, dim3(THREADS), 0, s, a);
  else if (unit == 8) launch_pdl(keep_rows_kernel<uint2>, grid, dim3(THREADS), 0, s, a);
  else if (unit == 4) launch_pdl(keep_rows_kernel<unsigned>, grid, dim3(THREADS), 0, s, a);
  else if (unit == 2) launch_pdl(keep_rows_kernel<unsigned short>, grid, dim3(THREADS), 0, s, a);
  else launch_pdl(keep_rows_kernel<unsigned char>, grid, dim3(THREADS), 0, s, a);
  return OMNIA_LAUNCH_RESULT();
}
