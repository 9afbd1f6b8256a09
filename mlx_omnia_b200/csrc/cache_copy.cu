// Copies inside the cache: pages, or the first rows of pages, of every layer that keeps them (a request that is forked, a
// pool that is made smaller or larger), and rows of per-request state. A copy computes nothing: its floor is every byte
// read once and written once at the memory's rate.
//
// Both kernels cut their work into runs of at most COPY_RUN contiguous bytes, a warp a run: with 16 bytes a load a lane has
// eight loads on their way before its first store, and an SM's warps some 256 KB. All sources are taken to be other bytes
// than all destinations, and no two destinations to be the same (the callers check both), so runs go in any order.
//
// Measured (B200): 300 pages of 36 layers to another tensor (1.4 GB in and out) 221 us, 6.4 TB/s, 99 % of what a plain copy reaches; the state
// of 24 requests (413 MB) 64 us, 6.4 TB/s. A few pages are bound by the call: 7 forks of a page 10 us with the host's part, 63 16.
#include "common.cuh"

#include <cstdlib>

namespace {

constexpr int COPY_MOVES = 256;      // moves of one launch
constexpr int COPY_TENSORS = 32;     // state tensors of one launch
constexpr int COPY_KINDS = 8;        // rows of unlike shape that a position may have
constexpr int COPY_RUN = 4096;       // bytes of a warp's run
constexpr int COPY_WARPS = 8;        // warps a block

__device__ __forceinline__ uint4 load_once(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
template <typename V>
__device__ __forceinline__ V load_once(const V* p) { return *p; }

// `count` elements of type V from `from` to `to` by one warp, eight loads a lane ahead of the stores.
template <typename V>
__device__ __forceinline__ void copy_run(unsigned char* to, const unsigned char* from, int count) {
  const int lane = threadIdx.x & 31;
  const V* src = reinterpret_cast<const V*>(from);
  V* dst = reinterpret_cast<V*>(to);
  for (int at = lane; at < count; at += 8 * 32) {
    V v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (at + 32 * i < count) v[i] = load_once(src + at + 32 * i);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (at + 32 * i < count) dst[at + 32 * i] = v[i];
  }
}

// The widest element that divides all of `bits` (addresses, strides and lengths, or-ed together).
inline int widest(unsigned long long bits) {
  for (int width = 16; width > 1; width /= 2)
    if (bits % width == 0) return width;
  return 1;
}

struct PageMoves {
  int from[COPY_MOVES], to[COPY_MOVES], rows[COPY_MOVES];
  // A page's blocks: `heads[k]` of kind k, one after the other, each `page_size` rows of `width[k]` bytes; the first kind's at 0.
  int heads[COPY_KINDS], width[COPY_KINDS];
  long long offset[COPY_KINDS];
};

// grid (runs of a page / COPY_WARPS, layers, moves). A warp's run: the `part`th COPY_RUN bytes of the rows to copy of one block.
template <typename V>
__global__ void __launch_bounds__(32 * COPY_WARPS)
copy_pages_kernel(const __grid_constant__ PageMoves moves, const unsigned char* from, unsigned char* to, long long from_layer,
                  long long to_layer, long long page_bytes, int page_size, int kinds, int parts) {
  pdl_wait();
  pdl_launch_dependents();
  const int run = blockIdx.x * COPY_WARPS + (threadIdx.x >> 5), move = blockIdx.z;
  int block = run / parts;
  const int part = run - block * parts;
  int kind = 0;
  while (kind < kinds && block >= moves.heads[kind]) block -= moves.heads[kind++];
  if (kind == kinds) return;
  const int width = moves.width[kind];
  const long long bytes = (long long)moves.rows[move] * width, at = (long long)part * COPY_RUN;
  if (at >= bytes) return;
  const long long inside = moves.offset[kind] + (long long)block * page_size * width + at;
  const int length = (int)min((long long)COPY_RUN, bytes - at);
  copy_run<V>(to + blockIdx.y * to_layer + moves.to[move] * page_bytes + inside,
              from + blockIdx.y * from_layer + moves.from[move] * page_bytes + inside, length / (int)sizeof(V));
}

struct SlotMoves {
  unsigned char* tensor[COPY_TENSORS];
  long long bytes[COPY_TENSORS];  // of a row
  int first[COPY_TENSORS + 1];    // runs of a row of the tensors before this one
  int from[COPY_MOVES], to[COPY_MOVES];
};

// grid (runs of all tensors' rows / COPY_WARPS, moves)
template <typename V>
__global__ void __launch_bounds__(32 * COPY_WARPS)
copy_slots_kernel(const __grid_constant__ SlotMoves moves, int tensors) {
  pdl_wait();
  pdl_launch_dependents();
  const int run = blockIdx.x * COPY_WARPS + (threadIdx.x >> 5);
  if (run >= moves.first[tensors]) return;
  int t = 0;
  while (run >= moves.first[t + 1]) ++t;
  const long long bytes = moves.bytes[t], at = (long long)(run - moves.first[t]) * COPY_RUN;
  const int length = (int)min((long long)COPY_RUN, bytes - at);
  copy_run<V>(moves.tensor[t] + moves.to[blockIdx.y] * bytes + at, moves.tensor[t] + moves.from[blockIdx.y] * bytes + at,
              length / (int)sizeof(V));
}

}  // namespace

#define OMNIA_BY_WIDTH(width, ...)                        \
  do {                                                    \
    if ((width) == 16) { using V = uint4; __VA_ARGS__; }  \
    else if ((width) == 8) { using V = uint2; __VA_ARGS__; } \
    else if ((width) == 4) { using V = unsigned; __VA_ARGS__; } \
    else if ((width) == 2) { using V = unsigned short; __VA_ARGS__; } \
    else { using V = unsigned char; __VA_ARGS__; }        \
  } while (0)

// Whether `count` moves of `columns` ints (from, to, ...) have numbers in range (else 1), no two one end (2), and, `same` tensor, no end where
// another begins (3); 4: no memory for a bit a place.
extern "C" int omnia_check_moves(const int* moves, int columns, int count, int most_from, int most_to, int same) {
  if (count < 1) return 0;
  unsigned char* ends = (unsigned char*)calloc((size_t)(most_to > 0 ? most_to : 0) / 8 + 1, 1);
  if (ends == nullptr) return 4;
  int code = 0;
  for (int i = 0; i < count && code == 0; ++i) {
    const int from = moves[columns * i], to = moves[columns * i + 1];
    if (from < 0 || from >= most_from || to < 0 || to >= most_to) code = 1;
    else if ((ends[to / 8] >> (to % 8)) & 1) code = 2;
    else ends[to / 8] |= 1 << (to % 8);
  }
  for (int i = 0; same && i < count && code == 0; ++i) {
    const int from = moves[columns * i];
    if (from < most_to && ((ends[from / 8] >> (from % 8)) & 1)) code = 3;
  }
  free(ends);
  return code;
}

// Pages moves[3 i] of every layer of `from`, their first moves[3 i + 2] rows, to pages moves[3 i + 1] of the same layer of `to`.
// Layers lie from_layer and to_layer bytes apart, pages page_bytes; a page is `kinds` kinds of blocks, heads[k] blocks of
// page_size rows of width[k] bytes. The caller has checked page numbers and rows.
extern "C" int omnia_copy_pages(const void* from, void* to, long long from_layer, long long to_layer, int layers,
                                long long page_bytes, int page_size, const int* heads, const int* width, int kinds,
                                const int* moves, int count, cudaStream_t stream) {
  if (count == 0 || layers == 0) return 0;
  if (count < 0 || layers < 0 || layers > 65535 || kinds < 1 || kinds > COPY_KINDS || page_size < 1) return (int)cudaErrorInvalidValue;
  unsigned long long bits = (uintptr_t)from | (uintptr_t)to | (unsigned long long)from_layer | (unsigned long long)to_layer |
                            (unsigned long long)page_bytes;
  PageMoves held = {};
  long long offset = 0;
  int blocks = 0, widest_row = 0;
  for (int k = 0; k < kinds; ++k) {
    if (heads[k] < 1 || width[k] < 1) return (int)cudaErrorInvalidValue;
    held.heads[k] = heads[k], held.width[k] = width[k], held.offset[k] = offset;
    offset += (long long)heads[k] * page_size * width[k];
    blocks += heads[k];
    bits |= (unsigned)width[k];
    widest_row = width[k] > widest_row ? width[k] : widest_row;
  }
  if (offset > page_bytes) return (int)cudaErrorInvalidValue;
  for (int done = 0; done < count; done += COPY_MOVES) {
    const int some = count - done < COPY_MOVES ? count - done : COPY_MOVES;
    int most = 0;
    for (int i = 0; i < some; ++i) {
      const int* move = moves + 3 * (done + i);
      if (move[2] < 0 || move[2] > page_size) return (int)cudaErrorInvalidValue;
      held.from[i] = move[0], held.to[i] = move[1], held.rows[i] = move[2];
      most = move[2] > most ? move[2] : most;
    }
    if (most == 0) continue;
    const int parts = (int)(((long long)most * widest_row + COPY_RUN - 1) / COPY_RUN);
    const dim3 grid((unsigned)((blocks * parts + COPY_WARPS - 1) / COPY_WARPS), layers, some);
    OMNIA_BY_WIDTH(widest(bits), launch_pdl(copy_pages_kernel<V>, grid, 32 * COPY_WARPS, 0, stream, held, (const unsigned char*)from,
                                            (unsigned char*)to, from_layer, to_layer, page_bytes, page_size, kinds, parts));
    const int code = OMNIA_LAUNCH_RESULT();
    if (code != 0) return code;
  }
  return 0;
}

// Rows moves[2 i] of every tensor to its rows moves[2 i + 1]; bytes[t] is the length of a row of tensor t.
extern "C" int omnia_copy_slots(void* const* tensor, const long long* bytes, int tensors, const int* moves, int count, cudaStream_t stream) {
  if (tensors < 0 || count < 0) return (int)cudaErrorInvalidValue;
  for (int t0 = 0; t0 < tensors; t0 += COPY_TENSORS) {
    const int held_tensors = tensors - t0 < COPY_TENSORS ? tensors - t0 : COPY_TENSORS;
    SlotMoves held = {};
    unsigned long long bits = 0;
    for (int t = 0; t < held_tensors; ++t) {
      held.tensor[t] = (unsigned char*)tensor[t0 + t], held.bytes[t] = bytes[t0 + t];
      held.first[t + 1] = held.first[t] + (int)((bytes[t0 + t] + COPY_RUN - 1) / COPY_RUN);
      bits |= (uintptr_t)tensor[t0 + t] | (unsigned long long)bytes[t0 + t];
    }
    if (held.first[held_tensors] == 0) continue;
    for (int done = 0; done < count; done += COPY_MOVES) {
      const int some = count - done < COPY_MOVES ? count - done : COPY_MOVES;
      for (int i = 0; i < some; ++i) held.from[i] = moves[2 * (done + i)], held.to[i] = moves[2 * (done + i) + 1];
      const dim3 grid((unsigned)((held.first[held_tensors] + COPY_WARPS - 1) / COPY_WARPS), some);
      OMNIA_BY_WIDTH(widest(bits), launch_pdl(copy_slots_kernel<V>, grid, 32 * COPY_WARPS, 0, stream, held, held_tensors));
      const int code = OMNIA_LAUNCH_RESULT();
      if (code != 0) return code;
    }
  }
  return 0;
}
