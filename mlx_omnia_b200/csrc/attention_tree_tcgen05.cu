// Attention of trees of drafted tokens in bfloat16 on the 5th-generation tensor cores, for requests that bring many rows. Compiled for one head size:
//   -DHEAD_DIM=64|128
//
// Floor: a request's keys and values once (4 D bytes a position and key/value head) at the memory's rate, or the products' 4 D operations a row and
// position, whichever is more; 256 rows are where the two meet.
//
// Measured, 32 / 8 heads of 128: 32 requests of up to 8,192 positions with up to 64 tokens (795 MB, 0.14 PFLOP) 298 us, 325 as the GPU gets to its power limit
// (1,000 W, 1.97 -> 1.79 GHz), 0.47 PFLOP/s, 2.7 TB/s; 4 of up to 131,072 with up to 24 (1.49 GB) 268, 300 to 330 at the limit (1.49 GHz), 4.5 to 5.6 TB/s.
// 16 / 8 heads, 8 of up to 4,096 with up to 16 (100 MB): 40.5, of which 12 to 15 are beginnings, ends and the join. What bounds the first is a tile's chain:
// 5,700 cycles for 128 keys of 256 rows, 2.9 us at 1.97 GHz where the products alone would take 1.5; 79 tiles an SM are 230 us, the rest the
// beginnings and ends of an SM's two to four segments. Of the 2,850 cycles that a softmax warp has for a half, 330 go to whether the scores are there, 170 to their load, 370 to the maximum, 330 to the offset,
// 1,350 to weights, sums and pairs (707 without the exponentials), 320 to the store. For every instruction issued 0.94 warps wait for one to be fetched: code
// taken out of the loop, though never run, is gained. Float32 in pairs and maxima of three: 1,030 for the weights, the same time in all. Error against
// 64 bits 0.0023 of the outputs' size, where a 32-bit form rounded once has 0.0017.
//
// A block has an SM and an equal share of the step's tiles of 128 keys (TreeShares), and works it off item by item: up to 256 rows (node, query
// head of the group) of one request and key/value head, in two slots of 128 that are two softmax chains. Each slot has a score tile of 128
// columns and an accumulator in tensor memory, a warp that issues its products and four warps of a thread a row, and works on halves of 64 keys:
//   S = Q K^T   tcgen05.mma (M 128, N 64) over the head size, while the half before is weighted
//   softmax     a row's 64 scores in registers at once; P takes the scores' place, rounded to bfloat16 as the product with V wants it (the
//               sum is of what was not rounded); the exponent's offset follows a row's maximum lazily
//   O += P V    tcgen05.mma (M 128, N head size), P read from tensor memory
// With more than 128 rows a slot has half of them and both see every tile; with fewer both hold the same rows and take the tiles in turn, and the
// two states are brought together at the item's end. The rows of a request's nodes follow one another, so one box of TMA brings a slot's queries.
// Keys and values come by TMA, a box of 16 keys x 64 dims, into rings of stages of 64 keys; numbering and tiles begin at multiples of 16.
//
// What a row does not see: where a half has nodes, the edge of a window or the end of the keys, a row's scores are taken through its bits. A value
// that is no finite number would reach every row there (0 x NaN is NaN), so such a half's values are looked through, and if there is one, the
// half's product is summed by hand, row by row, over what each row sees.
#ifndef HEAD_DIM
#define HEAD_DIM 128
#endif

#include "attention_tcgen05.cuh"
#include "attention_tree.cuh"
namespace {

constexpr int D = HEAD_DIM;
static_assert(D == 64 || D == 128, "head sizes 64 and 128");
constexpr int DH = D / 64;               // 64-wide halves of a head
constexpr int BAR_BYTES = 768;           // of shared memory, for two sets of barriers and the words behind them
constexpr int EXTRA = 5;                 // tiles that an item's beginning and end cost
constexpr int BM = 128, BN = 128, HALF = 64;  // rows of a slot, keys of a tile, of the halves that are worked on
// Seven tiles of shared memory: the rows (one tile where both slots hold the same, else two), the rest in stages of half a tile, as many for keys
// as for values: five each that both slots read, or three each a slot where the slots take turns with the tiles.
constexpr int TILES = 7, OWN_STAGES = 3, BOTH_STAGES = 5, MOST_STAGES = 2 * OWN_STAGES;
constexpr int SOFTMAX_THREADS = 256;     // warps 0-3 slot 0, 4-7 slot 1
constexpr int WARP_MMA = 8, WARP_K = 10, WARP_V = 12, WARP_Q = 14, WARP_INIT = 15, FEEDERS = 2;  // one issuer a slot; two warps feed each ring in turns
constexpr int THREADS = 512;
// Registers a thread, by warpgroup: the slots' softmax holds a row's 64 scores and the pairs made of them. Together they are what the block is launched with.
constexpr int SLOT_REGS = 192, OTHER_REGS = 64;
static_assert(2 * SLOT_REGS + 2 * OTHER_REGS == 4 * (65536 / THREADS), "a register split's sum is the launch's");
constexpr uint32_t HALF_BYTES = 128 * 128;   // 128 rows of 128 bytes
constexpr uint32_t TILE_BYTES = DH * HALF_BYTES;
constexpr uint32_t BOX_BYTES = 16 * 128;     // 16 keys x 64 dims
constexpr uint32_t SIDE_BYTES = HALF * 128, STAGE_BYTES = DH * SIDE_BYTES;  // of half a tile of keys or values
static_assert(TILE_BYTES + 2 * MOST_STAGES * STAGE_BYTES <= TILES * TILE_BYTES && 2 * TILE_BYTES + 2 * BOTH_STAGES * STAGE_BYTES <= TILES * TILE_BYTES,
              "rows and stages fit");
static_assert((TREE_MOST_REQUESTS + THREADS / 32) * sizeof(long long) <= TILES * TILE_BYTES, "the requests' ends lie where the tiles are to be");
constexpr uint32_t TMEM_COLS = 512, O_COL = 2 * BN;  // two score tiles, then two accumulators

// mbar_wait without a time to sleep for: a warp that asks for one wakes up later.
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  if (omnia_mbar_test(bar, parity)) return true;
  for (uint32_t i = 0; i < WAIT_LIMIT; ++i) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    if (done) return true;
    if ((i & 63) == 63 && *abort_flag) return false;
  }
  *abort_flag = 1;
  return false;
}
// Whether three barriers' phases are complete: bits 0, 1, 2. A question takes some 300 cycles to be answered, so they are asked together.
__device__ __forceinline__ uint32_t ask_three(uint32_t bar0, uint32_t parity0, uint32_t bar1, uint32_t parity1, uint32_t bar2, uint32_t parity2) {
  uint32_t a, b, c;
  asm volatile(
      "{\n\t.reg .pred p, q, r;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%3], %4;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 q, [%5], %6;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 r, [%7], %8;\n\t"
      "selp.u32 %0, 1, 0, p;\n\tselp.u32 %1, 2, 0, q;\n\tselp.u32 %2, 4, 0, r;\n\t}"
      : "=r"(a), "=r"(b), "=r"(c)
      : "r"(bar0), "r"(parity0), "r"(bar1), "r"(parity1), "r"(bar2), "r"(parity2)
      : "memory");
  return a | b | c;
}
__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 1, %0;" ::"n"(SOFTMAX_THREADS) : "memory"); }
__device__ __forceinline__ void block_sync() { asm volatile("bar.sync 0, %0;" ::"n"(THREADS) : "memory"); }
__device__ __forceinline__ void mbar_inval(uint32_t bar) { asm volatile("mbarrier.inval.shared::cta.b64 [%0];" ::"r"(bar) : "memory"); }

// A row's bits for the 64 nodes from m0 on (which may be below 0: bits of keys that are held, none here).
__device__ __forceinline__ uint32_t node_bits(const int* row, int words, int m) {
  const int w = m >> 5, by = m & 31;
  const uint32_t lo = w >= 0 && w < words ? (uint32_t)row[w] : 0u, hi = w + 1 >= 0 && w + 1 < words ? (uint32_t)row[w + 1] : 0u;
  return by ? (lo >> by) | (hi << (32 - by)) : lo;
}
__device__ __forceinline__ bool no_number(uint32_t pair) { return (pair & 0x7f80u) == 0x7f80u || (pair & 0x7f800000u) == 0x7f800000u; }

// What a block does next: some tiles of an item. It lies in shared memory, made by one warp between two segments.
struct Segment {
  TreeKeys k;
  int request, kvh, row0, rows, lo, hi;  // lo, hi: keys, as numbered; rows 0: nothing more
  bool whole, turns;
};
constexpr int TAIL_BYTES = 4 * BM * sizeof(float) + 2 * (sizeof(Segment) + 15) / 16 * 16;

}  // namespace

// CAPPED: with a cap on the scores. (A kernel of its own: 300 instructions in the middle of a loop that is bound by fetching them, 2 % of long steps.)
template <bool CAPPED>
__global__ void __launch_bounds__(THREADS, 1)
tree_tcgen05_kernel(const __grid_constant__ CUtensorMap map_kv, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ TreeAttention a,
                    const TreeShares shares) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  if (smem_u32(smem_raw) & 1023u) {  // the swizzled tiles need a base on 1024 bytes
    if (threadIdx.x == 0) atomicOr(a.err, OMNIA_ERR_TIMEOUT);
    return;
  }
  unsigned char* q_s = smem_raw;
  uint64_t* bars = reinterpret_cast<uint64_t*>(q_s + TILES * TILE_BYTES);
  // bars: q_full | k_full[] | k_empty[] | v_full[] | v_empty[] | s_full[2][2] | p_full[2][2] | o_done[2][2] (slot, half) | began; a set of them for
  // every other segment, so that one is made while the other is in use
  constexpr int BARS = 1 + 4 * MOST_STAGES + 13;
  static_assert(2 * BARS * 8 + 24 <= BAR_BYTES, "barriers and the words behind them");
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + 2 * BARS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  volatile int* by_hand = reinterpret_cast<volatile int*>(tmem_holder + 2);  // [2][2]: whether a slot's half has been summed without a product
  float* row_ml = reinterpret_cast<float*>(reinterpret_cast<unsigned char*>(bars) + BAR_BYTES);  // [2][128][2]: a slot's offset and sum, for the other one
  Segment* segments = reinterpret_cast<Segment*>(row_ml + 4 * BM);
  const int warp = omnia_warp_index(), lane = threadIdx.x & 31;
  constexpr uint32_t K_FULL = 8, K_EMPTY = K_FULL + 8 * MOST_STAGES, V_FULL = K_EMPTY + 8 * MOST_STAGES, V_EMPTY = V_FULL + 8 * MOST_STAGES,
                     S_FULL = V_EMPTY + 8 * MOST_STAGES, P_FULL = S_FULL + 32, O_DONE = P_FULL + 32, BEGAN = O_DONE + 32;
  if (warp == WARP_MMA) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)), "r"(TMEM_COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_kv) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_q) : "memory");
  }
  // From here on what earlier kernels wrote is read; the launch is a programmatic dependent one.
  pdl_wait();
  pdl_launch_dependents();
  long long* ends = reinterpret_cast<long long*>(smem_raw);
  const long long total = shares.lay_out(a, ends, ends + TREE_MOST_REQUESTS);
  const long long blocks = min((long long)gridDim.x, total);
  TreePlace place;  // (one warp's)
  place.left = 0;
  const long long upto = blocks ? total * (blockIdx.x + 1) / blocks : 0;
  if (blockIdx.x < blocks && warp == WARP_INIT) {
    const long long t0 = total * blockIdx.x / blocks;
    place.find(a, shares, ends, t0, (int)(upto - t0));
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // (the ends lie where copies will come to)
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = *tmem_holder;
  OMNIA_TRACE_BLOCK(2);  // the shares are known
  const int group = a.nq / a.nkv, slot_nodes = BM / group, slot_rows = slot_nodes * group;

  int stages = 1, issued = -1;  // of a ring; the last half tile that this warp has asked for
  uint32_t k_at = 0, v_at = 0;  // byte offsets of the rings in shared memory
  const Segment* now = segments;
  // A slot's sequence of half tiles: half u is the (u & 1)th of the tile j0 + (u >> 1) * step.
  auto halves_of = [&](int j0) {
    const int tiles = (now->hi - now->lo + BN - 1) / BN, step = now->turns ? 2 : 1;
    const int mine = tiles > j0 ? (tiles - j0 + step - 1) / step : 0, last = j0 + (mine - 1) * step;
    return mine < 1 ? 0 : 2 * mine - (now->hi - now->lo - last * BN <= HALF ? 1 : 0);
  };
  auto first_of = [&](int j0, int u) { return now->lo + (j0 + (u >> 1) * (now->turns ? 2 : 1)) * BN + (u & 1) * HALF; };  // its first key
  // Half u's stage, and the parity of the phase in which it is full.
  auto stage_of = [&](int slot, int u) { return (now->turns ? slot * OWN_STAGES : 0) + u % stages; };
  auto phase_of = [&](int u) { return (u / stages) & 1; };
  // All warps go from segment to segment side by side. One of them makes the next, and its barriers, while the others are at work.
  int turn_of = -1;  // segments begun, less one
  auto make_segment = [&](int which) {  // (a lane of the one warp)
    Segment& n = segments[which & 1];
    n.rows = 0;
    if (place.left == 0) return;
    const int tiles = min(place.tiles - place.tile, place.left);
    n.k = place.k, n.request = place.request, n.kvh = place.head;
    n.row0 = place.row_tile * shares.rows;
    n.lo = place.tile * BN, n.hi = min((place.tile + tiles) * BN, place.k.total);
    const int rows = min(shares.rows, place.k.count * group - n.row0);
    n.whole = tiles == place.tiles, n.turns = rows <= slot_rows;
    if (place.tile == 0) tree_note(a, total, blocks, upto, place, which == 0);
    place.next(a, shares, tiles);
    const uint32_t set = smem_u32(bars) + (which & 1) * BARS * 8;
    if (which > 1)
      for (int i = 0; i < BARS; ++i) mbar_inval(set + 8 * i);
    const int readers = n.turns ? 1 : 2;
    mbar_init(set, 1);
    for (int i = 0; i < MOST_STAGES; ++i) mbar_init(set + K_FULL + 8 * i, 1), mbar_init(set + K_EMPTY + 8 * i, readers);
    for (int i = 0; i < MOST_STAGES; ++i) mbar_init(set + V_FULL + 8 * i, 1), mbar_init(set + V_EMPTY + 8 * i, readers);
    for (int i = 0; i < 4; ++i) mbar_init(set + S_FULL + 8 * i, 1), mbar_init(set + P_FULL + 8 * i, BM / 32), mbar_init(set + O_DONE + 8 * i, 1);
    mbar_init(set + BEGAN, BM / 32);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    n.rows = rows;
  };
  if (warp == WARP_INIT && lane == 0) {
    for (int i = 0; i < 4; ++i) by_hand[i] = 0;
    make_segment(0);
  }
  uint32_t q_full = 0, k_full0 = 0, k_empty0 = 0, v_full0 = 0, v_empty0 = 0, s_full0 = 0, p_full0 = 0, o_done0 = 0, began = 0;
  auto next_segment = [&]() {  // -> whether there is one
    block_sync();  // all are done with the one before
    ++turn_of;
    if (segments[turn_of & 1].rows == 0 || *abort_flag) return false;
    issued = -1;
    const bool turns = segments[turn_of & 1].turns;
    stages = turns ? OWN_STAGES : BOTH_STAGES;
    k_at = (turns ? 1 : 2) * TILE_BYTES;
    v_at = k_at + (turns ? MOST_STAGES : BOTH_STAGES) * STAGE_BYTES;
    q_full = smem_u32(bars) + (turn_of & 1) * BARS * 8;
    k_full0 = q_full + K_FULL, k_empty0 = q_full + K_EMPTY, v_full0 = q_full + V_FULL, v_empty0 = q_full + V_EMPTY;
    s_full0 = q_full + S_FULL, p_full0 = q_full + P_FULL, o_done0 = q_full + O_DONE, began = q_full + BEGAN;
    return true;
  };

  if (warp >= WARP_MMA) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OTHER_REGS));
  else asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SLOT_REGS));
  if (warp >= WARP_MMA) {
    while (next_segment()) {
      const Segment& s = segments[turn_of & 1];
      now = &s;
      const int tiles = (s.hi - s.lo + BN - 1) / BN;
      if (warp == WARP_Q) {
        // ---- the rows' queries, a box the group's heads of a slot's nodes x 64 dims. The rows behind the last node are other requests' or zeros: no
        // other row learns of them. ------------------------------------------------------------------------------------------------------
        if (omnia_elect_one()) {
          const int slots = s.turns ? 1 : 2;
          mbar_expect_tx(q_full, slots * slot_rows * DH * 128);
          for (int slot = 0; slot < slots; ++slot)
#pragma unroll
            for (int half = 0; half < DH; ++half)
              tma_load_3d(smem_u32(q_s) + slot * TILE_BYTES + half * HALF_BYTES, &map_q, q_full, half * 64, s.kvh * group,
                          s.k.first + s.row0 / group + slot * slot_nodes);
        }
        __syncwarp();
      } else if (warp >= WARP_K && warp < WARP_Q) {
        // ---- producers: two warps a ring, one a slot or taking turns; a lane looks up a box's page, one lane asks for the boxes ----
        const int which = warp >= WARP_V ? 1 : 0, turn = warp - (which ? WARP_V : WARP_K), j0 = s.turns ? turn : 0, halves = halves_of(j0);
        const int* table = a.block_table + (size_t)s.request * a.max_pages;
        const uint32_t full0 = which ? v_full0 : k_full0, empty0 = which ? v_empty0 : k_empty0;
        const int u0 = s.turns ? 0 : turn, du = s.turns ? 1 : FEEDERS;
        auto lookup = [&](int u, int& key) {  // the page of this lane's 16 keys of half u (-2: none that the segment reads), the first of these
          const int x = first_of(j0, u) + lane * 16;
          key = s.k.key(x);
          if (lane >= HALF / 16 || u >= halves || x >= s.hi) return -2;
          const int at = key / a.page_size;
          return at < a.max_pages ? table[at] : -1;
        };
        bool ok = true;
        int key_cur, key_next, page_cur = lookup(u0, key_cur);
        for (int u = u0; u < halves; u += du) {
          const int page_next = lookup(u + du, key_next), st = stage_of(turn, u);
          if (lane == 0 && u >= stages) ok = wait_for(empty0 + 8 * st, phase_of(u) ^ 1, abort_flag);
          ok = __shfl_sync(0xffffffffu, ok, 0);
          if (!ok) break;
          bool load = page_cur != -2;
          if (load && (page_cur < 0 || page_cur >= a.num_pages)) atomicOr(a.err, OMNIA_ERR_PAGE), load = false;
          const uint32_t loaded = __ballot_sync(0xffffffffu, load);
          const int mine = load ? ((page_cur * 2 + which) * a.nkv + s.kvh) * a.page_size + key_cur % a.page_size : 0;
          int y[HALF / 16];
#pragma unroll
          for (int x = 0; x < HALF / 16; ++x) y[x] = __shfl_sync(0xffffffffu, mine, x);
          if (omnia_elect_one()) {
            mbar_expect_tx(full0 + 8 * st, __popc(loaded) * DH * BOX_BYTES);
            const uint32_t dst = smem_u32(q_s + (which ? v_at : k_at) + st * STAGE_BYTES);
#pragma unroll
            for (int x = 0; x < HALF / 16; ++x)
              if ((loaded >> x) & 1u)
#pragma unroll
                for (int side = 0; side < DH; ++side)
                  tma_load_2d(dst + side * SIDE_BYTES + x * BOX_BYTES, &map_kv, full0 + 8 * st, side * 64, y[x]);
          }
          __syncwarp();
          issued = u;
          page_cur = page_next, key_cur = key_next;
        }
      } else if (warp == WARP_INIT) {
        if (lane == 0) make_segment(turn_of + 1);
        __syncwarp();
      } else if (warp < WARP_K) {
        // ---- issuer of a slot's products -------------------------------------------------------------------------------
        const int slot = warp - WARP_MMA, j0 = s.turns ? slot : 0, halves = halves_of(j0);
        if (halves > 0 && omnia_elect_one()) {
          constexpr uint32_t instr_s = idesc(BM, HALF, false), instr_o = idesc(BM, D, true);
          const uint64_t q_desc = desc_k_major(smem_u32(q_s + (s.turns ? 0 : slot) * TILE_BYTES));
          const uint32_t s_tmem = tmem_base + slot * BN, o_tmem = tmem_base + O_COL + slot * D;
          uint32_t accumulate = 0;
          bool ok = wait_for(q_full, 0, abort_flag);
          // The second slot begins when the first one's first weights are there: its exponentials then run while the other one's products do, and
          // not beside the other one's exponentials.
          if (slot == 1 && tiles > 1 && ok) ok = wait_for(began, 0, abort_flag);
          // Stages are counted on, not divided out: this thread's instructions are what the slot's chain waits for.
          const int base = s.turns ? slot * OWN_STAGES : 0;
          int k_st = base, v_st = base;
          uint32_t k_ph = 0, v_ph = 0;
          auto scores = [&](int h, bool there) {  // of the next half; `there`: its keys have been seen to be
            ok = there || wait_for(k_full0 + 8 * k_st, k_ph, abort_flag);
            if (!ok) return;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint64_t k_desc = desc_k_major(smem_u32(q_s + k_at + k_st * STAGE_BYTES));
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
              umma(s_tmem + h * HALF, q_desc + (((kk / 4) * HALF_BYTES + (kk % 4) * 32) >> 4),
                   k_desc + (((kk / 4) * SIDE_BYTES + (kk % 4) * 32) >> 4), instr_s, kk != 0);
            umma_commit(s_full0 + 8 * (2 * slot + h));
            umma_commit(k_empty0 + 8 * k_st);
            if (++k_st == base + stages) k_st = base, k_ph ^= 1;
          };
          if (ok) scores(0, false);
          if (ok && halves > 1) scores(1, false);
          for (int u = 0; u < halves && ok; ++u) {
            const int h = u & 1;
            const uint32_t t = (u >> 1) & 1, p_full = p_full0 + 8 * (2 * slot + h), o_done = o_done0 + 8 * (2 * slot + h);
            const uint32_t there = ask_three(p_full, t, v_full0 + 8 * v_st, v_ph, k_full0 + 8 * k_st, k_ph);
            ok = ((there & 2) || wait_for(v_full0 + 8 * v_st, v_ph, abort_flag)) && ((there & 1) || wait_for(p_full, t, abort_flag));
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (by_hand[2 * slot + h]) {
              by_hand[2 * slot + h] = 0;  // (the slot's warps write it again two halves on, behind products that come behind this)
              accumulate = 1;
            } else {
              const uint64_t v_desc = desc_mn_major(smem_u32(q_s + v_at + v_st * STAGE_BYTES), SIDE_BYTES);
              // Boxes that were loaded: the rest of the stage, of a last half, is stale.
              const int boxes = u + 1 < halves ? HALF / 16 : min(HALF, s.hi - first_of(j0, u) + 15) / 16;
#pragma unroll
              for (int kk = 0; kk < HALF / 16; ++kk) {
                if (kk >= boxes) break;
                // P: 16 keys are eight columns of packed pairs
                umma_ts(o_tmem, s_tmem + h * HALF + kk * 8, v_desc + ((kk * BOX_BYTES) >> 4), instr_o, accumulate);
                accumulate = 1;
              }
            }
            umma_commit(o_done);
            umma_commit(v_empty0 + 8 * v_st);
            if (++v_st == base + stages) v_st = base, v_ph ^= 1;
            // The half's columns are free once its weights have been read.
            if (u + 2 < halves) {
              ok = wait_for(o_done, t, abort_flag);
              if (ok) scores(h, there & 4);
            }
          }
        }
        __syncwarp();
        // The set is made anew behind this segment, so whatever this slot's products tell a barrier has to have been told: the stages that they read
        // last and the accumulator's last two halves, a lane a barrier. (What else arrives, another warp of the segment has waited for.)
        const int back = lane & 7, last = halves - 1 - back;
        if (last >= 0 && back < (lane < 16 ? stages : lane < 24 ? 2 : 0)) {
          const uint32_t bar = lane < 16 ? (lane < 8 ? k_empty0 : v_empty0) + 8 * stage_of(slot, last) : o_done0 + 8 * (2 * slot + (last & 1));
          wait_for(bar, lane < 16 ? phase_of(last) : (last >> 1) & 1, abort_flag);
        }
        __syncwarp();
      }
    }
  } else {
    // ---- softmax: a thread a row of its slot -----------------------------------------------------------------------------
    const int slot = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lane_field = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_addr = tmem_base + lane_field + slot * BN, o_addr = tmem_base + lane_field + O_COL + slot * D;
    const float cap = a.softcap * LOG2E, twice = CAPPED ? 2.f * a.scale / a.softcap * LOG2E : 0.f, unit = CAPPED ? 1.f : a.scale * LOG2E;
    bool first = true;
    while (next_segment()) {
      const Segment& s = segments[turn_of & 1];
      now = &s;
      const int my_row = s.turns ? row : slot * slot_rows + row;   // among the segment's rows
      const bool live = row < slot_rows && my_row < s.rows;
      const int node = live ? (s.row0 + my_row) / group : 0, pos = a.positions[s.k.first + node], low = tree_low(a, pos);
      const int* sees = a.ancestors + (size_t)(s.k.first + node) * a.words;
      const int clear_from = tree_low(a, s.k.held + s.k.count - 1);  // what no row's window ends above
      OMNIA_TRACE_BLOCK(3);  // a segment begins
      float m = -INFINITY, l = 0.f;  // the row's offset (log2 units), its sum against it
      bool ok = true;
      int done = 0;
      // The turn ahead of a block's first tile works on whatever tensor memory holds, and leaves it in the accumulator, which the first product
      // overwrites: it fetches the code, a straight line of some thousand instructions that every launch finds cold, while the first
      // tile is on its way.
      const int j0 = s.turns ? slot : 0, halves = halves_of(j0);
      for (int u = halves > 0 && first ? -1 : 0; u < halves; ++u) {
        const bool dry = u < 0;
        const int h = dry ? 0 : u & 1, t = u >> 1;
        const uint32_t half_addr = s_addr + h * HALF;
        const int x0 = dry ? 0 : first_of(j0, u), seen = dry ? HALF : min(HALF, s.hi - x0);  // keys of this half; the columns beyond hold whatever the stage held
        const bool clear = dry || (seen == HALF && x0 >= s.k.kept && s.k.key(x0) >= clear_from && s.k.key(x0 + HALF - 1) < s.k.held);
        // What a row sees of a half that not all rows see all of, and whether one of its values is no number: asked for ahead of the scores.
        uint32_t bits[2] = {~0u, ~0u};
        bool odd = false;
        if (!clear) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int x = x0 + 32 * i, ends_at = s.hi - x;  // keys of these 32 that there are
            uint32_t b;
            if (a.window > 0 || a.run > 0) {
              b = 0;
#pragma unroll 1
              for (int c = 0; c < 32; ++c) {
                const int key = s.k.key(x + c), which = key - s.k.held;
                if (x + c >= s.hi) break;
                const int at = which < 0 ? key : a.positions[s.k.first + which];
                const bool near = at >= low || (a.window > 0 && at < a.keep);
                if (near && (which < 0 || (((uint32_t)sees[which >> 5] >> (which & 31)) & 1u))) b |= 1u << c;
              }
            } else {
              const int held = s.k.held - x;  // of these 32, how many are held
              b = (held >= 32 ? ~0u : held > 0 ? (1u << held) - 1u : 0u) | (held < 32 ? node_bits(sees, a.words, -held) : 0u);
            }
            bits[i] = ends_at >= 32 ? b : ends_at > 0 ? b & ((1u << ends_at) - 1u) : 0u;
          }
          const int st = stage_of(slot, u);
          ok = __all_sync(0xffffffffu, wait_for(v_full0 + 8 * st, phase_of(u), abort_flag));
          if (!ok) break;
          const unsigned char* v = q_s + v_at + st * STAGE_BYTES;
#pragma unroll
          for (int side = 0; side < DH; ++side)
#pragma unroll 4
            for (int i = lane; i < seen * 8; i += 32) {
              const uint4 x = *reinterpret_cast<const uint4*>(v + side * SIDE_BYTES + i * 16);
              odd |= no_number(x.x) | no_number(x.y) | no_number(x.z) | no_number(x.w);
            }
          odd = __any_sync(0xffffffffu, odd);  // (the same for all of the slot's warps: the stage is what it is)
        }
        if (!dry) {
          ok = __all_sync(0xffffffffu, wait_for(s_full0 + 8 * (2 * slot + h), t & 1, abort_flag));
          if (!ok) break;
          if (u == 0) OMNIA_TRACE_BLOCK(4);  // its first scores
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        // All of the row's scores at once: a load from tensor memory takes some 0.35 us to arrive.
        float z[HALF];
        {
          uint32_t raw[HALF];
#pragma unroll
          for (int c = 0; c < HALF; c += 32) tmem_load32(half_addr + c, raw + c);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
          for (int c = 0; c < HALF; ++c) z[c] = __uint_as_float(raw[c]);
        }
        if constexpr (CAPPED) {  // c tanh(x) = c - 2 c / (1 + e^2x), in log2 units (a score that is infinite has the cap, of its sign)
#pragma unroll
          for (int c = 0; c < HALF; ++c) z[c] = fmaf(-2.f * cap, fast_rcp(1.f + fast_exp2(z[c] * twice)), cap);
        }
        if (!clear) {
#pragma unroll
          for (int c = 0; c < HALF; ++c) z[c] = (bits[c / 32] >> (c % 32)) & 1u ? z[c] : -INFINITY;
        }
        float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < HALF; ++c) tops[c & 3] = fmaxf(tops[c & 3], z[c]);
        const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * unit;
        // The offset follows the row's maximum lazily: what was summed is brought to a new one only when the scores have outgrown the old.
        float alpha = 1.f;
        if (top > m) {
          if (m == -INFINITY) {
            m = top;
          } else if (top - m > RESCALE_STEP) {
            alpha = fast_exp2(m - top);
            l *= alpha;
            m = top;
          }
        }
        if (done > 0 && (odd || __any_sync(0xffffffffu, alpha != 1.f))) {
          // The products so far, the half before this one's among them, have to be done; the next one's wait for this warp.
          ok = __all_sync(0xffffffffu, wait_for(o_done0 + 8 * (2 * slot + (h ^ 1)), ((u - 1) >> 1) & 1, abort_flag));
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          if (__any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll 1
            for (int c = 0; c < D; c += 8) {
              uint32_t o[8];
              tmem_load8(o_addr + c, o);
              asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
              for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_store8(o_addr + c, o);
            }
          }
        }
        const float offset = m == -INFINITY ? 0.f : m;
        float sums[4] = {0.f, 0.f, 0.f, 0.f};
        // The weights, in pairs, take the place of the first half of these scores.
        uint32_t packed[HALF / 2];
#pragma unroll
        for (int c = 0; c < HALF; c += 2) {
          const float p0 = fast_exp2(fmaf(z[c], unit, -offset)), p1 = fast_exp2(fmaf(z[c + 1], unit, -offset));
          sums[c & 2] += p0, sums[(c & 2) + 1] += p1;
          packed[c / 2] = pack_bf16(p0, p1);
        }
        tmem_store32(dry ? o_addr : half_addr, packed);
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        if (dry) {
          m = -INFINITY, l = 0.f;
          continue;
        }
        l += (sums[0] + sums[1]) + (sums[2] + sums[3]);
        if (odd) {
          // The half by hand: a row's own sums over the keys that have a weight, eight dims and sixteen keys at a time.
          const unsigned char* v = q_s + v_at + stage_of(slot, u) * STAGE_BYTES;
#pragma unroll 1
          for (int c = 0; c < D; c += 8) {
            uint32_t o[8];
            if (done > 0) {
              tmem_load8(o_addr + c, o);
              asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            } else {
#pragma unroll
              for (int i = 0; i < 8; ++i) o[i] = 0u;
            }
#pragma unroll 1
            for (int k0 = 0; k0 < seen; k0 += 16) {
              uint32_t pairs[8];
              tmem_load8(half_addr + k0 / 2, pairs);
              asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll 1
              for (int k = 0; k < 16; ++k) {
                uint32_t two = pairs[0];
#pragma unroll
                for (int i = 1; i < 8; ++i) two = k / 2 == i ? pairs[i] : two;
                const float p = __uint_as_float(k & 1 ? two & 0xffff0000u : two << 16);
                if (k0 + k < seen && p != 0.f) {
                  const uint4 x = *reinterpret_cast<const uint4*>(v + c / 64 * SIDE_BYTES + (k0 + k) * 128 + ((c / 8 % 8) ^ (k & 7)) * 16);
                  const uint32_t values[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                  for (int i = 0; i < 8; ++i)
                    o[i] = __float_as_uint(fmaf(p, __uint_as_float(i & 1 ? values[i / 2] & 0xffff0000u : values[i / 2] << 16), __uint_as_float(o[i])));
                }
              }
            }
            tmem_store8(o_addr + c, o);
          }
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          by_hand[2 * slot + h] = 1;
        } else if (seen & 15) {
          // The last box reaches past the last key. Its rows of V beyond get no weight, but what they hold need not be a number
          // (0 x NaN is NaN): they are cleared once the stage has landed, by both slots where both read it.
          const int st = stage_of(slot, u), r1 = (seen + 15) & ~15;
#pragma unroll 1
          for (int i = row; i < (r1 - seen) * DH * 8; i += BM) {
            const int piece = i & 7, side = (i >> 3) % DH, r = seen + (i >> 3) / DH;
            *reinterpret_cast<uint4*>(q_s + v_at + st * STAGE_BYTES + side * SIDE_BYTES + r * 128 + piece * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(p_full0 + 8 * (2 * slot + h));
          if (u == 0 && slot == 0) mbar_arrive(began);
        }
        ++done;
      }
      // ---- the segment's end: offset, sum, accumulator. The accumulators' rows go through shared memory (all of it but the barriers: both slots'
      // products are done behind the first barrier, and every load has landed, since products have read it), so that a warp writes a row at a time. ----
      if (ok && done > 0) ok = __all_sync(0xffffffffu, wait_for(o_done0 + 8 * (2 * slot + ((done - 1) & 1)), ((done - 1) >> 1) & 1, abort_flag));
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      OMNIA_TRACE_BLOCK(5);  // its last product
      constexpr int STRIDE = D + 4;  // floats: eight lanes' 16 bytes lie in different banks
      float* stage = reinterpret_cast<float*>(smem_raw) + (s.turns ? 0 : slot) * BM * STRIDE;
      static_assert(2 * BM * STRIDE * sizeof(float) <= TILES * TILE_BYTES, "both slots' rows fit where the tiles were");
      float both = m, w = 1.f;  // of a row whose two slots' states become one: the offset, and what this slot's state counts
      if (s.turns) row_ml[(slot * BM + row) * 2] = m, row_ml[(slot * BM + row) * 2 + 1] = l;
      softmax_sync();
      if (s.turns) {
        const float other_m = row_ml[((slot ^ 1) * BM + row) * 2], other_l = row_ml[((slot ^ 1) * BM + row) * 2 + 1];
        both = fmaxf(m, other_m);
        w = m == -INFINITY ? 0.f : fast_exp2(m - both);
        l = l * w + other_l * (other_m == -INFINITY ? 0.f : fast_exp2(other_m - both));  // (a sum that is no number stays none)
      }
      const size_t part = (2 * (size_t)blockIdx.x + (first ? 0 : 1)) * shares.rows;
      if (ok && live && !s.whole && (!s.turns || slot == 0)) a.part_ml[2 * (part + my_row)] = both, a.part_ml[2 * (part + my_row) + 1] = l;
      if (s.whole) {  // the answer: against the sink, by the sum
        const float sink = a.sink && live ? a.sink[s.kvh * group + (s.row0 + my_row) % group] * LOG2E : -INFINITY;
        const float over = fmaxf(both, sink), offset = over == -INFINITY ? 0.f : over, f = fast_exp2(both - offset);
        const float all = l * f + fast_exp2(sink - offset);
        w = all > 0.f || all != all ? w * f / all : 0.f;
      }
      // This slot's rows, weighted, to the stage; where the rows are both slots', the second slot's first.
      auto put_rows = [&](bool add) {
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
          if (done > 0) {
            tmem_load32(o_addr + c, o);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
          }
          float4* to = reinterpret_cast<float4*>(stage + row * STRIDE + c);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float4 y = add ? to[i] : make_float4(0.f, 0.f, 0.f, 0.f);
            if (done > 0 && w != 0.f) {  // (a slot without a tile has nothing in its accumulator)
              y.x = fmaf(__uint_as_float(o[4 * i]), w, y.x), y.y = fmaf(__uint_as_float(o[4 * i + 1]), w, y.y);
              y.z = fmaf(__uint_as_float(o[4 * i + 2]), w, y.z), y.w = fmaf(__uint_as_float(o[4 * i + 3]), w, y.w);
            }
            to[i] = y;
          }
        }
      };
      if (s.turns) {
        if (slot == 1) put_rows(false);
        softmax_sync();
        if (slot == 0) put_rows(true);
        softmax_sync();
      } else {
        put_rows(false);
        __syncwarp();
      }
      // Rows out: a warp's own 32, or 16 of the rows that were both slots'.
      const int r0 = s.turns ? warp * 16 : quarter * 32, r1 = min(r0 + (s.turns ? 16 : 32), min(slot_rows, s.rows - (s.turns ? 0 : slot * slot_rows)));
      const int row_at = s.turns ? 0 : slot * slot_rows;
      const bool mine = ok && lane < D / 4;
      if (!s.whole) {
#pragma unroll 4
        for (int r = r0; r < r1; ++r)
          if (mine) reinterpret_cast<float4*>(a.part_o + (part + row_at + r) * D)[lane] = reinterpret_cast<const float4*>(stage + r * STRIDE)[lane];
      } else {
        // A lane knows where the row that is as many behind the warp's first one goes.
        const int at = s.row0 + row_at + min(r0 + lane, r1 - 1), my_token = s.k.first + at / group, my_head = s.kvh * group + at % group;
        const bool pairs = ((reinterpret_cast<uintptr_t>(a.gate) | (uintptr_t)a.gate_stride * 2) & 7) == 0;
#pragma unroll 1
        for (int r = r0; r < r1; r += 4) {  // (four rows' gates on their way at once)
          uint2 gates[4];
          int tokens[4], heads[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            tokens[i] = __shfl_sync(0xffffffffu, my_token, r - r0 + i), heads[i] = __shfl_sync(0xffffffffu, my_head, r - r0 + i);
            if (a.gate && mine) {
              const bf16* gate = static_cast<const bf16*>(a.gate) + (size_t)tokens[i] * a.gate_stride + heads[i] * D + 4 * lane;
              if (pairs) {
                gates[i] = *reinterpret_cast<const uint2*>(gate);
              } else {
                const unsigned short* g = reinterpret_cast<const unsigned short*>(gate);
                gates[i] = make_uint2(g[0] | (uint32_t)g[1] << 16, g[2] | (uint32_t)g[3] << 16);
              }
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (!mine || r + i >= r1) continue;
            float4 y = reinterpret_cast<const float4*>(stage + (r + i) * STRIDE)[lane];
            if (a.gate) {
              y.x *= tree_sigmoid(__uint_as_float(gates[i].x << 16)), y.y *= tree_sigmoid(__uint_as_float(gates[i].x & 0xffff0000u));
              y.z *= tree_sigmoid(__uint_as_float(gates[i].y << 16)), y.w *= tree_sigmoid(__uint_as_float(gates[i].y & 0xffff0000u));
            }
            *reinterpret_cast<uint2*>(static_cast<bf16*>(a.out) + ((size_t)tokens[i] * a.nq + heads[i]) * D + 4 * lane) =
                make_uint2(pack_bf16(y.x, y.y), pack_bf16(y.z, y.w));
          }
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // (the rows lay where the next segment's copies come to)
      OMNIA_TRACE_BLOCK(6);  // its rows are out
      first = false;
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (*abort_flag && warp >= WARP_K && warp < WARP_Q && lane == 0) {
    // Given up: what this warp has asked for must land before the block's shared memory goes away. (Its last copies, one a stage; a
    // stage that the ring's other warp has filled since reads as not complete, so the wait is short.)
    const uint32_t full0 = warp >= WARP_V ? v_full0 : k_full0;
    const int turn = warp - (warp >= WARP_V ? WARP_V : WARP_K);
    for (int u = issued; u >= 0 && u > issued - stages; u -= now->turns ? 1 : FEEDERS)
      for (uint32_t i = 0; i < WAIT_LIMIT / 1024 && !mbar_try(full0 + 8 * stage_of(turn, u), phase_of(u)); ++i) {
      }
  }
  if (*abort_flag && warp == WARP_Q && lane == 0 && q_full != 0)
    for (uint32_t i = 0; i < WAIT_LIMIT / 1024 && !mbar_try(q_full, 0); ++i) {
    }
  if (warp == WARP_MMA) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS));
  if (threadIdx.x == 0 && *abort_flag) atomicOr(a.err, OMNIA_ERR_TIMEOUT);
}

namespace {

template <bool CAPPED>
int launch(const CUtensorMap& map_kv, const CUtensorMap& map_q, const TreeAttention& a, const TreeShares& shares, int blocks, cudaStream_t stream) {
  constexpr size_t smem = TILES * (size_t)TILE_BYTES + BAR_BYTES + TAIL_BYTES;
  static bool configured[64] = {};
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return (int)cudaErrorInvalidDevice;
  if (!configured[device]) {
    const cudaError_t e = cudaFuncSetAttribute(tree_tcgen05_kernel<CAPPED>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return (int)e;
    configured[device] = true;
  }
  return (int)launch_pdl(tree_tcgen05_kernel<CAPPED>, dim3(blocks), THREADS, smem, stream, map_kv, map_q, a, shares);
}

}  // namespace

// Pages [num_pages, 2, nkv, page_size, D], page_size a multiple of 16; q [tokens, nq, D]. `blocks`: what the work is shared out over, an SM each, with
// two slots of `omnia_tree_tcgen05_rows` rows in part_o and part_ml.
extern "C" int omnia_tree_tcgen05_rows(int group) { return 2 * (BM / group * group); }

extern "C" int omnia_tree_attention_tcgen05(const TreeAttention* given, int most_nodes, int blocks, cudaStream_t stream) {
  TreeAttention a = *given;
  const int group = a.nkv > 0 ? a.nq / a.nkv : 0;
  if (a.requests < 1 || a.requests > TREE_MOST_REQUESTS || group < 1 || group > BM || a.nq != a.nkv * group || a.nkv > 65535 || a.d != D || a.dv != D ||
      a.page_size < 16 || a.page_size % 16 || a.max_pages < 1 || a.num_pages < 1 || ((uintptr_t)a.q & 15) || ((uintptr_t)a.k_pages & 15) ||
      ((uintptr_t)a.part_o & 15) || a.softcap < 0.f || a.scale <= 0.f || blocks < 1 || most_nodes < 1 || a.page_stride != 2LL * a.nkv * a.page_size * D ||
      (long long)a.num_pages * 2 * a.nkv * a.page_size > 0x7fffffffLL)
    return (int)cudaErrorInvalidValue;
  EncodeTiled encode = encode_tiled();
  if (encode == nullptr) return (int)cudaErrorNotSupported;
  CUtensorMap map_kv, map_q;
  const cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)a.num_pages * 2 * a.nkv * a.page_size};
  const cuuint64_t strides[1] = {(cuuint64_t)D * 2};
  const cuuint32_t box[2] = {64, 16}, elem[3] = {1, 1, 1};
  if (encode(&map_kv, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(a.k_pages), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return (int)cudaErrorInvalidValue;
  // Queries [tokens, nq, D]: a box is the group's heads of a slot's nodes x 64 dims.
  const cuuint64_t q_dims[3] = {(cuuint64_t)D, (cuuint64_t)a.nq, (cuuint64_t)a.tokens};
  const cuuint64_t q_strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)a.nq * D * 2};
  const cuuint32_t q_box[3] = {64, (cuuint32_t)group, (cuuint32_t)(BM / group)};
  if (encode(&map_q, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(a.q), q_dims, q_strides, q_box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return (int)cudaErrorInvalidValue;
  const TreeShares shares = {omnia_tree_tcgen05_rows(group), BN, 16, EXTRA};
  a.parts = tree_row_tiles(a, most_nodes, shares.rows);
  const int code = a.softcap > 0.f ? launch<true>(map_kv, map_q, a, shares, blocks, stream) : launch<false>(map_kv, map_q, a, shares, blocks, stream);
  if (code) return code;
  return tree_join<bf16, D>(a, shares, most_nodes, blocks, stream);
}
