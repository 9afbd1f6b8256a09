// What the kernels of attention over shared positions are handed (attention_shared.cu, which says what they compute;
// attention_shared_tc.cu; attention_tc.cu compiled with -DSHARED=1).
#pragma once
#include "common.cuh"

// The list `plan` holds, ints: starts[requests] (the positions that a request shares), parts[requests] (the
// pieces that these were cut into), members[...] (request numbers, group by group), then `items` of ITEM_INTS ints:
// (request whose pages are read, place of the group's first member in `members`, first row, rows, key/value head, first key,
// last key + 1, piece); rows < 1: nothing to do.
constexpr int SHARED_ITEM_INTS = 8;

struct SharedAttention {
  const void *q, *k_pages, *v_pages, *gate;
  void* out;
  const int *block_table, *cu_seqlens, *seq_lens, *plan;
  const float* sink;
  float *part_o, *part_ml;
  int* err;
  long long page_stride;
  int requests, members, items, max_parts, chunk_keys, max_chunks, gate_stride, max_pages, num_pages, nq, nkv, d, dv, page_size, maps;
  float scale, softcap;
  MapDifference difference;
};
