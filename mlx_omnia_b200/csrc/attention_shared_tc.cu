// The shared positions of attention_shared.cu in bfloat16 on the 5th-generation tensor cores: a group's keys and values are
// fetched once and attended to by the rows of all its requests. Compiled for one head size and one group size:
//   -DHEAD_DIM=64|128   -DGROUP=g (query heads per key/value head, g <= 16)
//
// Floor: the shared keys and values once (4 D bytes a position and key/value head) at the memory's rate, or the
// products' 4 D operations a row and position, whichever is more: 256 rows are where the two meet.
//
// A block has an SM, one key/value head, one run of keys (an item of the list) and up to 256 rows, in two slots of 128, which are two
// softmax chains that know nothing of one another: each has a score tile of 128 columns and an accumulator in tensor memory, a
// warp that issues its products and four warps of a thread a row. A slot works on halves of 64 keys, two of which have their columns:
//   S = Q K^T   tcgen05.mma (M 128, N 64) over the head size, while the half before is weighted
//   softmax     a row's 64 scores in registers at once; P takes the scores' place, rounded to bfloat16 as the product with V wants it (the
//               sum is of what was not rounded; outputs are off by 0.0023 of their size, where rounding them alone gives 0.0017);
//               the exponent's offset follows a row's maximum lazily, and only then is the accumulator rescaled
//   O += P V    tcgen05.mma (M 128, N head size), P read from tensor memory
// One chain alone would wait for its own products and loads half of the time; two fill each other's gaps. With more
// than 128 rows a slot has half of them and both see every tile of keys; with fewer both hold the same rows and take the tiles
// in turn, and the two states are brought together at the end. The rows are gathered from wherever the requests' tokens lie, by TMA.
// Keys and values come by TMA, a box of 16 keys x 64 dims, into rings of stages of 64 keys.
//
// Measured (B200, 32/8 heads of 128): 64 requests of 65,536 shared positions and up to 1,024 of their own, with the decode kernel beside,
// 117 us a layer (floor 68, memory; each request for itself 2,600); 96 of 30,000 + 64 83 us (floor 28, memory; products 48), 16 of
// 32,768 + 500 45 (24). A tile of 128 keys takes a block 2.3 to 2.6 us with 256 rows. Of that the products take 1.8: a step of 16 dims is 76
// cycles where it scores 64 keys and 102 where it scores 128, since its 128 rows come out of shared memory each time, a step of 16 keys of
// the second product 52 to 77. Whole tiles of 128 keys have the cheaper scores but wait for them between two softmaxes: 3.3 us. The
// softmax itself has room (exponentials' unit 55 %, schedulers 56 % on the busiest SM): two teams of warps a slot, one a half, made it slower (96 of 30,000: 84 us,
// so 91), and so did asking for the next half's scores ahead of this one's exponentials (96).
#ifndef HEAD_DIM
#define HEAD_DIM 128
#endif
#ifndef GROUP
#define GROUP 2
#endif

#include "attention_tcgen05.cuh"
#include "attention_shared.cuh"
namespace {

constexpr int D = HEAD_DIM;
static_assert(D == 64 || D == 128, "head sizes 64 and 128");
static_assert(GROUP >= 1 && GROUP <= 16, "group size must be 1..16");
constexpr int DH = D / 64;               // 64-wide halves of a head
constexpr int BAR_BYTES = 384;           // of shared memory, for barriers
constexpr int BM = 128, BN = 128, HALF = 64;  // rows of a slot, keys of a tile, of the halves that are worked on
constexpr int SLOT_ROWS = BM / GROUP * GROUP;
// Seven tiles of shared memory: the rows (one tile where both slots hold the same, else two), the rest in stages of a half tile, as many for keys
// as for values: five each that both slots read, or, where the slots take turns with the tiles, three each a slot, of its own halves: a stage
// that both used in turns would complete a phase which the slower slot has yet to wait for. (Whole tiles, four stages for keys and two for
// values, left a slot that takes turns one stage of values, asked for when the weights were already on their way: 16 requests of 32,768
// positions 45.3 us, so 44.6; 4 of 65,536 63.5 and 59.0.)
constexpr int TILES = 7, OWN_STAGES = 3, BOTH_STAGES = 5, MOST_STAGES = 2 * OWN_STAGES;
constexpr int SOFTMAX_THREADS = 256;     // warps 0-3 slot 0, 4-7 slot 1
constexpr int SLOT_MEMBERS = BM / GROUP, Q_MEMBERS = 8;  // requests of a slot's rows, of a box of queries
constexpr int WARP_MMA = 8, WARP_K = 10, WARP_V = 12, WARP_Q = 14, FEEDERS = 2;  // one issuer a slot; two warps feed each ring in turns
constexpr int THREADS = 512;             // (a warp has nothing to do)
// Registers a thread, by warpgroup: the slots' softmax holds a row's 64 scores and the pairs made of them. Together they are what the block is launched with.
constexpr int SLOT_REGS = 192, OTHER_REGS = 64;
static_assert(2 * SLOT_REGS + 2 * OTHER_REGS == 4 * (65536 / THREADS), "a register split's sum is the launch's");
constexpr uint32_t HALF_BYTES = 128 * 128;   // 128 rows of 128 bytes
constexpr uint32_t TILE_BYTES = DH * HALF_BYTES;
constexpr uint32_t BOX_BYTES = 16 * 128;     // 16 keys x 64 dims
constexpr uint32_t SIDE_BYTES = HALF * 128, STAGE_BYTES = DH * SIDE_BYTES;  // of half a tile of keys or values
static_assert(TILE_BYTES + 2 * MOST_STAGES * STAGE_BYTES <= TILES * TILE_BYTES && 2 * TILE_BYTES + 2 * BOTH_STAGES * STAGE_BYTES <= TILES * TILE_BYTES,
              "rows and stages fit");
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
__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 1, %0;" ::"n"(SOFTMAX_THREADS) : "memory"); }

}  // namespace

__global__ void __launch_bounds__(THREADS, 1)
shared_pieces_tc_kernel(const __grid_constant__ CUtensorMap map_kv, const __grid_constant__ CUtensorMap map_q,
                        const __grid_constant__ CUtensorMap map_q8, const __grid_constant__ SharedAttention a) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  if (smem_u32(smem_raw) & 1023u) {  // the swizzled tiles need a base on 1024 bytes
    if (threadIdx.x == 0) atomicOr(a.err, OMNIA_ERR_TIMEOUT);
    return;
  }
  unsigned char* q_s = smem_raw;
  uint64_t* bars = reinterpret_cast<uint64_t*>(q_s + TILES * TILE_BYTES);
  // bars: q_full | k_full[] | k_empty[] | v_full[] | v_empty[] | s_full[2][2] | p_full[2][2] | o_done[2][2] (slot, half) | began
  constexpr int BARS = 1 + 4 * MOST_STAGES + 13;
  static_assert(BARS * 8 + 8 <= BAR_BYTES, "barriers and the two words behind them");
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + BARS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  float* row_ml = reinterpret_cast<float*>(tmem_holder + 2);  // [2][128][2]: a slot's offset and sum, for the other one
  const int warp = omnia_warp_index(), lane = threadIdx.x & 31;
  const uint32_t q_full = smem_u32(bars), k_full0 = q_full + 8, k_empty0 = k_full0 + 8 * MOST_STAGES, v_full0 = k_empty0 + 8 * MOST_STAGES,
                 v_empty0 = v_full0 + 8 * MOST_STAGES, s_full0 = v_empty0 + 8 * MOST_STAGES, p_full0 = s_full0 + 32, o_done0 = p_full0 + 32,
                 began = o_done0 + 32;
  if (warp == WARP_MMA) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)), "r"(TMEM_COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  // From here on what earlier kernels wrote is read; the launch is a programmatic dependent one.
  pdl_wait();
  pdl_launch_dependents();
  const int *members = a.plan + 2 * a.requests, *item = members + a.members + SHARED_ITEM_INTS * blockIdx.x;
  const int table_of = item[0], first_member = item[1], row0 = item[2], rows = item[3], kvh = item[4], lo = item[5], hi = item[6], part = item[7];
  const bool turns = rows <= SLOT_ROWS;           // both slots hold the same rows and take the tiles in turn
  const int stages = turns ? OWN_STAGES : BOTH_STAGES;  // of a ring
  unsigned char* k_s = q_s + (turns ? 1 : 2) * TILE_BYTES;
  unsigned char* v_s = k_s + (turns ? MOST_STAGES : BOTH_STAGES) * STAGE_BYTES;
  const int tiles = rows < 1 ? 0 : (hi - lo + BN - 1) / BN;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    const int readers = turns ? 1 : 2;
    for (int s = 0; s < MOST_STAGES; ++s) mbar_init(k_full0 + 8 * s, 1), mbar_init(k_empty0 + 8 * s, readers);
    for (int s = 0; s < MOST_STAGES; ++s) mbar_init(v_full0 + 8 * s, 1), mbar_init(v_empty0 + 8 * s, readers);
    for (int s = 0; s < 4; ++s) mbar_init(s_full0 + 8 * s, 1), mbar_init(p_full0 + 8 * s, BM / 32), mbar_init(o_done0 + 8 * s, 1);
    mbar_init(began, BM / 32);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = *tmem_holder;
  int issued = -1;  // the last half tile that this warp has asked for
  // A slot's sequence of half tiles: half u is the (u & 1)th of the tile j0 + (u >> 1) * step.
  const int step = turns ? 2 : 1;
  auto halves_of = [&](int j0) {
    const int mine = tiles > j0 ? (tiles - j0 + step - 1) / step : 0, last = j0 + (mine - 1) * step;
    return mine < 1 ? 0 : 2 * mine - (hi - lo - last * BN <= HALF ? 1 : 0);
  };
  auto first_of = [&](int j0, int u) { return lo + (j0 + (u >> 1) * step) * BN + (u & 1) * HALF; };  // its first key
  // Half u's stage, and the parity of the phase in which it is full.
  auto stage_of = [&](int slot, int u) { return (turns ? slot * OWN_STAGES : 0) + u % stages; };
  auto phase_of = [&](int u) { return (u / stages) & 1; };

  if (warp >= WARP_MMA) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OTHER_REGS));
  if (warp > WARP_Q) {
    // (nothing)
  } else if (warp == WARP_Q) {
    // ---- the rows' queries, a box the group's rows of a request x 64 dims, or of eight requests that are neighbours in the step (a box takes its
    // issuer 40 ns). The rows of a tile that hold nothing are whatever was there: no other row learns of it. --------------------------------
    const int count = rows / GROUP, first = first_member + row0 / GROUP;
    if (tiles > 0) {
      if (omnia_elect_one()) mbar_expect_tx(q_full, rows * DH * 128);
      __syncwarp();
      for (int m0 = 0; m0 < count; m0 += 32) {
        const int some = min(32, count - m0), mine = lane < some ? a.cu_seqlens[members[first + m0 + lane]] : -1;  // tokens
        const uint32_t follow = __ballot_sync(0xffffffffu, __shfl_down_sync(0xffffffffu, mine, 1) == mine + 1 && lane + 1 < some);
        constexpr uint32_t ALL = (1u << (Q_MEMBERS - 1)) - 1;
        for (int m = 0; m < some;) {
          const int token = __shfl_sync(0xffffffffu, mine, m), member = m0 + m, slot = member / SLOT_MEMBERS, at = member % SLOT_MEMBERS;
          const bool eight = m + Q_MEMBERS <= some && at + Q_MEMBERS <= SLOT_MEMBERS && ((follow >> m) & ALL) == ALL;
          if (omnia_elect_one())
#pragma unroll
            for (int half = 0; half < DH; ++half)
              tma_load_3d(smem_u32(q_s) + slot * TILE_BYTES + half * HALF_BYTES + at * GROUP * 128, eight ? &map_q8 : &map_q, q_full, half * 64,
                          kvh * GROUP, token);
          __syncwarp();
          m += eight ? Q_MEMBERS : 1;
        }
      }
    }
  } else if (warp >= WARP_K) {
    // ---- producers: two warps a ring, one a slot or taking turns; a lane looks up a box's page, one lane asks for the boxes ----
    const int which = warp >= WARP_V ? 1 : 0, turn = warp - (which ? WARP_V : WARP_K), j0 = turns ? turn : 0, halves = halves_of(j0);
    const int* table = a.block_table + (size_t)table_of * a.max_pages;
    const uint32_t full0 = which ? v_full0 : k_full0, empty0 = which ? v_empty0 : k_empty0;
    const int u0 = turns ? 0 : turn, du = turns ? 1 : FEEDERS;
    auto lookup = [&](int u) {  // the page of this lane's 16 keys of half u (-2: none that the item reads)
      const int pos = first_of(j0, u) + lane * 16;
      return lane < HALF / 16 && u < halves && pos < hi ? table[pos / a.page_size] : -2;
    };
    bool ok = true;
    int page_cur = lookup(u0);
    for (int u = u0; u < halves; u += du) {
      const int page_next = lookup(u + du), s = stage_of(turn, u), pos = first_of(j0, u) + lane * 16;
      if (lane == 0 && u >= stages) ok = wait_for(empty0 + 8 * s, phase_of(u) ^ 1, abort_flag);
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok) break;
      bool load = page_cur != -2;
      if (load && (page_cur < 0 || page_cur >= a.num_pages)) atomicOr(a.err, OMNIA_ERR_PAGE), load = false;
      const uint32_t loaded = __ballot_sync(0xffffffffu, load);
      const int mine = load ? ((page_cur * 2 + which) * a.nkv + kvh) * a.page_size + pos % a.page_size : 0;
      int y[HALF / 16];
#pragma unroll
      for (int x = 0; x < HALF / 16; ++x) y[x] = __shfl_sync(0xffffffffu, mine, x);
      if (omnia_elect_one()) {
        mbar_expect_tx(full0 + 8 * s, __popc(loaded) * DH * BOX_BYTES);
        const uint32_t dst = smem_u32((which ? v_s : k_s) + s * STAGE_BYTES);
#pragma unroll
        for (int x = 0; x < HALF / 16; ++x)
          if ((loaded >> x) & 1u)
#pragma unroll
            for (int side = 0; side < DH; ++side)
              tma_load_2d(dst + side * SIDE_BYTES + x * BOX_BYTES, &map_kv, full0 + 8 * s, side * 64, y[x]);
      }
      __syncwarp();
      issued = u;
      page_cur = page_next;
    }
  } else if (warp >= WARP_MMA) {
    // ---- issuer of a slot's products -----------------------------------------------------------------------------------
    const int slot = warp - WARP_MMA, j0 = turns ? slot : 0, halves = halves_of(j0);
    if (halves > 0 && omnia_elect_one()) {
      constexpr uint32_t instr_s = idesc(BM, HALF, false), instr_o = idesc(BM, D, true);
      const uint64_t q_desc = desc_k_major(smem_u32(q_s + (turns ? 0 : slot) * TILE_BYTES));
      const uint32_t s_tmem = tmem_base + slot * BN, o_tmem = tmem_base + O_COL + slot * D;
      uint32_t accumulate = 0;
      bool ok = wait_for(q_full, 0, abort_flag);
      // The second slot begins when the first one's first weights are there: its exponentials then run while the other one's products do, and
      // not beside the other one's exponentials.
      if (slot == 1 && tiles > 1 && ok) ok = wait_for(began, 0, abort_flag);
      auto scores = [&](int u) {
        const int h = u & 1, s = stage_of(slot, u);
        ok = wait_for(k_full0 + 8 * s, phase_of(u), abort_flag);
        if (!ok) return;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint64_t k_desc = desc_k_major(smem_u32(k_s + s * STAGE_BYTES));
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          umma(s_tmem + h * HALF, q_desc + (((kk / 4) * HALF_BYTES + (kk % 4) * 32) >> 4), k_desc + (((kk / 4) * SIDE_BYTES + (kk % 4) * 32) >> 4),
               instr_s, kk != 0);
        umma_commit(s_full0 + 8 * (2 * slot + h));
        umma_commit(k_empty0 + 8 * s);
      };
      if (ok) scores(0);
      if (ok && halves > 1) scores(1);
      for (int u = 0; u < halves && ok; ++u) {
        const int h = u & 1, t = u >> 1, s = stage_of(slot, u);
        ok = wait_for(v_full0 + 8 * s, phase_of(u), abort_flag) && wait_for(p_full0 + 8 * (2 * slot + h), t & 1, abort_flag);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint64_t v_desc = desc_mn_major(smem_u32(v_s + s * STAGE_BYTES), SIDE_BYTES);
        const int groups = min(HALF, hi - first_of(j0, u) + 15) / 16;  // boxes that were loaded: the rest of the stage is stale
#pragma unroll
        for (int kk = 0; kk < HALF / 16; ++kk) {
          if (kk >= groups) break;
          // P: 16 keys are eight columns of packed pairs
          umma_ts(o_tmem, s_tmem + h * HALF + kk * 8, v_desc + ((kk * BOX_BYTES) >> 4), instr_o, accumulate);
          accumulate = 1;
        }
        umma_commit(o_done0 + 8 * (2 * slot + h));
        umma_commit(v_empty0 + 8 * s);
        // The half's columns are free once its weights have been read.
        if (u + 2 < halves) {
          ok = wait_for(o_done0 + 8 * (2 * slot + h), t & 1, abort_flag);
          if (ok) scores(u + 2);
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SLOT_REGS));
    // ---- softmax: a thread a row of its slot -----------------------------------------------------------------------------
    const int slot = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    auto place = [&](int r, int& request, int& head) {
      request = members[first_member + (row0 + r) / GROUP];
      head = kvh * GROUP + (row0 + r) % GROUP;
    };
    const int my_row = turns ? row : slot * SLOT_ROWS + row;   // among the item's rows
    const bool live = row < SLOT_ROWS && my_row < rows;
    const uint32_t lane_field = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_addr = tmem_base + lane_field + slot * BN, o_addr = tmem_base + lane_field + O_COL + slot * D;
    const bool capped = a.softcap > 0.f;
    const float cap = a.softcap * LOG2E, twice = capped ? 2.f * a.scale / a.softcap * LOG2E : 0.f, unit = capped ? 1.f : a.scale * LOG2E;
    float m = -INFINITY, l = 0.f;  // the row's offset (log2 units), its sum against it
    bool ok = true;
    int done = 0;
    // The turn ahead of the first tile works on whatever tensor memory holds, and leaves it in the accumulator, which the first product
    // overwrites: it fetches the code, a straight line of some thousand instructions that every launch finds cold, while the first
    // tile is on its way (without it a block's first tile took 3 us).
    const int j0 = turns ? slot : 0, halves = halves_of(j0);
    for (int u = halves > 0 ? -1 : 0; u < halves; ++u) {
      const bool dry = u < 0;
      const int h = dry ? 0 : u & 1, t = u >> 1;
      const uint32_t half_addr = s_addr + h * HALF;
      if (!dry) {
        ok = __all_sync(0xffffffffu, wait_for(s_full0 + 8 * (2 * slot + h), t & 1, abort_flag));
        if (!ok) break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const int seen = dry ? HALF : min(HALF, hi - first_of(j0, u));  // keys of this half; the columns beyond hold whatever the stage held
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
      if (capped) {  // c tanh(x) = c - 2 c / (1 + e^2x), in log2 units (a score that is infinite has the cap, of its sign)
#pragma unroll
        for (int c = 0; c < HALF; ++c) z[c] = fmaf(-2.f * cap, fast_rcp(1.f + fast_exp2(z[c] * twice)), cap);
      }
      if (seen < HALF) {
#pragma unroll
        for (int c = 0; c < HALF; ++c) z[c] = c < seen ? z[c] : -INFINITY;
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
      if (done > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
        // The products so far, the half before this one's among them, have to be done; the next one's wait for this warp.
        ok = __all_sync(0xffffffffu, wait_for(o_done0 + 8 * (2 * slot + (h ^ 1)), ((u - 1) >> 1) & 1, abort_flag));
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
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
      if (seen & 15) {
        // The last box reaches past the last key. Its rows of V beyond get no weight, but what they hold need not be a number
        // (0 x NaN is NaN): they are cleared once the stage has landed, by both slots where both read it.
        const int s = stage_of(slot, u);
        ok = __all_sync(0xffffffffu, wait_for(v_full0 + 8 * s, phase_of(u), abort_flag));
        if (!ok) break;
        const int r1 = (seen + 15) & ~15;
#pragma unroll 1
        for (int i = row; i < (r1 - seen) * DH * 8; i += BM) {
          const int piece = i & 7, side = (i >> 3) % DH, r = seen + (i >> 3) / DH;
          *reinterpret_cast<uint4*>(v_s + s * STAGE_BYTES + side * SIDE_BYTES + r * 128 + piece * 16) = make_uint4(0u, 0u, 0u, 0u);
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
    // ---- the slot's piece: offset, sum, accumulator. The accumulators' rows go through shared memory (all of it but the barriers: both slots'
    // products are done behind the first barrier, and every load has landed, since products have read it), so that a warp writes a row
    // of 512 bytes at a time: a thread a row wrote 16 bytes here and there, 3 us of a block's end and 8 where both slots have rows. -------
    if (ok && done > 0) ok = __all_sync(0xffffffffu, wait_for(o_done0 + 8 * (2 * slot + ((done - 1) & 1)), ((done - 1) >> 1) & 1, abort_flag));
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    constexpr int STRIDE = D + 4;  // floats: eight lanes' 16 bytes lie in different banks
    float* stage = reinterpret_cast<float*>(smem_raw) + (turns ? 0 : slot) * BM * STRIDE;
    static_assert(2 * BM * STRIDE * sizeof(float) <= TILES * TILE_BYTES, "both slots' rows fit where the tiles were");
    float both = m, w = 1.f;  // of a row whose two slots' states become one: the offset, and what this slot's state counts
    if (turns) row_ml[(slot * BM + row) * 2] = m, row_ml[(slot * BM + row) * 2 + 1] = l;
    softmax_sync();
    if (turns) {
      const float other_m = row_ml[((slot ^ 1) * BM + row) * 2], other_l = row_ml[((slot ^ 1) * BM + row) * 2 + 1];
      both = fmaxf(m, other_m);
      w = m == -INFINITY ? 0.f : fast_exp2(m - both);
      l = l * w + (other_m == -INFINITY ? 0.f : other_l * fast_exp2(other_m - both));
    }
    const int places = a.max_parts + a.max_chunks;
    auto place_of = [&](int r) {  // of row r of the item
      int request, head;
      place(r, request, head);
      return ((size_t)request * a.nq + head) * places + part;
    };
    if (ok && live && (!turns || slot == 0)) {
      const size_t at = place_of(my_row);
      a.part_ml[2 * at] = both, a.part_ml[2 * at + 1] = l;
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
          if (done > 0) {  // (a slot without a tile has nothing in its accumulator)
            y.x = fmaf(__uint_as_float(o[4 * i]), w, y.x), y.y = fmaf(__uint_as_float(o[4 * i + 1]), w, y.y);
            y.z = fmaf(__uint_as_float(o[4 * i + 2]), w, y.z), y.w = fmaf(__uint_as_float(o[4 * i + 3]), w, y.w);
          }
          to[i] = y;
        }
      }
    };
    if (turns) {
      if (slot == 1) put_rows(false);
      softmax_sync();
      if (slot == 0) put_rows(true);
      softmax_sync();
    } else {
      put_rows(false);
      __syncwarp();
    }
    // Rows out: a warp's own 32, or 16 of the rows that were both slots'.
    const int r0 = turns ? warp * 16 : quarter * 32, r1 = min(r0 + (turns ? 16 : 32), min(SLOT_ROWS, rows - (turns ? 0 : slot * SLOT_ROWS)));
#pragma unroll 4
    for (int r = r0; r < r1; ++r) {
      const size_t at = place_of((turns ? 0 : slot * SLOT_ROWS) + r);
      if (ok && lane < D / 4) reinterpret_cast<float4*>(a.part_o + at * D)[lane] = reinterpret_cast<const float4*>(stage + r * STRIDE)[lane];
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (*abort_flag && warp >= WARP_K && warp < WARP_Q && lane == 0) {
    // Given up: what this warp has asked for must land before the block's shared memory goes away. (Its last copies, one a stage; a
    // stage that the ring's other warp has filled since reads as not complete, so the wait is short.)
    const uint32_t full0 = warp >= WARP_V ? v_full0 : k_full0;
    const int turn = warp - (warp >= WARP_V ? WARP_V : WARP_K);
    for (int u = issued; u >= 0 && u > issued - stages; u -= turns ? 1 : FEEDERS)
      for (uint32_t i = 0; i < WAIT_LIMIT / 1024 && !mbar_try(full0 + 8 * stage_of(turn, u), phase_of(u)); ++i) {
      }
  }
  if (*abort_flag && warp == WARP_Q && lane == 0 && tiles > 0)
    for (uint32_t i = 0; i < WAIT_LIMIT / 1024 && !mbar_try(q_full, 0); ++i) {
    }
  if (warp == WARP_MMA) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS));
  if (threadIdx.x == 0 && *abort_flag) atomicOr(a.err, OMNIA_ERR_TIMEOUT);
}

// ---- the pieces of a request and key/value head, put together: grid (nkv, requests) --------------------------------------------
// A warp has a head's pieces, or every second, fourth, ... of them: eight maxima, sums and accumulators (16 bytes a lane) on their way at once. The
// group's heads (eight at a time) end side by side in shared memory, where the gate, or the difference of two maps, is taken.
constexpr int MERGE_WARPS = 8, MERGE_HEADS = GROUP < MERGE_WARPS ? GROUP : MERGE_WARPS, HEAD_WARPS = MERGE_WARPS / MERGE_HEADS;
__global__ void __launch_bounds__(32 * MERGE_WARPS)
shared_merge_tc_kernel(const __grid_constant__ SharedAttention a) {
  __shared__ __align__(16) float part[MERGE_HEADS][HEAD_WARPS][D];
  __shared__ float tops[MERGE_HEADS][HEAD_WARPS], sums[MERGE_HEADS][HEAD_WARPS];
  // The kernel before this one lets it begin only after its own wait for whatever came before, so lengths, list and gates are there.
  const int kvh = blockIdx.x, request = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int start = a.plan[request], parts = min(a.plan[a.requests + request], a.max_parts), pos = a.seq_lens[request] - 1;
  const size_t token = (size_t)a.cu_seqlens[request];
  constexpr int MINE = (MERGE_HEADS * D + 32 * MERGE_WARPS - 1) / (32 * MERGE_WARPS);
  float gates[MINE];
  auto ask_for_gates = [&](int h0) {
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      const int x = threadIdx.x + i * 32 * MERGE_WARPS;
      if (a.gate != nullptr && x < min(MERGE_HEADS, GROUP - h0) * D)
        gates[i] = __bfloat162float(((const bf16*)a.gate)[token * a.gate_stride + (size_t)(kvh * GROUP + h0) * D + x]);
    }
  };
  ask_for_gates(0);
  pdl_wait();
  pdl_launch_dependents();
  if (pos < 0) return;
  const int places = a.max_parts + a.max_chunks, pieces = parts + (pos < start ? 0 : min(pos / a.chunk_keys - start / a.chunk_keys + 1, a.max_chunks));
  for (int h0 = 0; h0 < GROUP; h0 += MERGE_HEADS) {
    if (h0 > 0) ask_for_gates(h0);
    const int h = warp / HEAD_WARPS, sub = warp % HEAD_WARPS, r = h0 + h;
    if (h < MERGE_HEADS && r < GROUP) {
      const size_t first = ((size_t)request * a.nq + kvh * GROUP + r) * places;
      float top = -INFINITY, l = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
      for (int p0 = sub; p0 < pieces; p0 += 8 * HEAD_WARPS) {
        float2 ml[8];
        float4 x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int p = p0 + u * HEAD_WARPS;
          ml[u] = make_float2(-INFINITY, 0.f), x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (p < pieces) {
            ml[u] = __ldcg(reinterpret_cast<const float2*>(a.part_ml) + first + p);
            if (lane < D / 4) x[u] = __ldcg(reinterpret_cast<const float4*>(a.part_o + (first + p) * D) + lane);
          }
        }
        float now = top;
#pragma unroll
        for (int u = 0; u < 8; ++u) now = fmaxf(now, ml[u].x);
        const float keep = top == -INFINITY ? 0.f : exp2f(top - now);
        l *= keep, acc.x *= keep, acc.y *= keep, acc.z *= keep, acc.w *= keep;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const float w = ml[u].x == -INFINITY ? 0.f : exp2f(ml[u].x - now);
          l = fmaf(ml[u].y, w, l);
          acc.x = fmaf(x[u].x, w, acc.x), acc.y = fmaf(x[u].y, w, acc.y), acc.z = fmaf(x[u].z, w, acc.z), acc.w = fmaf(x[u].w, w, acc.w);
        }
        top = now;
      }
      if (lane < D / 4) *reinterpret_cast<float4*>(&part[h][sub][4 * lane]) = acc;
      if (lane == 0) tops[h][sub] = top, sums[h][sub] = l;
    }
    __syncthreads();
    bf16* out = (bf16*)a.out;
    const int heads = min(MERGE_HEADS, GROUP - h0);
    auto value = [&](int h, int dim) {
      float top = -INFINITY, l = 0.f, v = 0.f;
#pragma unroll
      for (int x = 0; x < HEAD_WARPS; ++x) top = fmaxf(top, tops[h][x]);
      if (top == -INFINITY) return 0.f;  // nothing seen
#pragma unroll
      for (int x = 0; x < HEAD_WARPS; ++x) {
        const float w = tops[h][x] == -INFINITY ? 0.f : exp2f(tops[h][x] - top);
        l = fmaf(sums[h][x], w, l), v = fmaf(part[h][x][dim], w, v);
      }
      if (a.sink != nullptr) l += exp2f(a.sink[kvh * GROUP + h0 + h] * LOG2E - top);
      return v / l;
    };
    if (a.maps == 1) {
#pragma unroll
      for (int i = 0; i < MINE; ++i) {
        const int x = threadIdx.x + i * 32 * MERGE_WARPS;
        if (x >= heads * D) break;
        float y = value(x / D, x % D);
        if (a.gate != nullptr) y *= 1.f / (1.f + expf(-gates[i]));
        out[(token * a.nq + kvh * GROUP + h0) * D + x] = __float2bfloat16_rn(y);
      }
    } else if (2 * warp + 1 < heads) {  // a warp a pair of maps
      float d[D / 32], ss = 0.f;
#pragma unroll
      for (int k = 0; k < D / 32; ++k) {
        const int dim = lane + 32 * k;
        d[k] = dim < a.difference.dv ? value(2 * warp, dim) - a.difference.lambda * value(2 * warp + 1, dim) : 0.f;
        ss += d[k] * d[k];
      }
      const float f = rsqrtf(warp_sum(ss) / (float)a.difference.dv + a.difference.eps) * a.difference.factor;
#pragma unroll
      for (int k = 0; k < D / 32; ++k)
        if (lane + 32 * k < a.difference.dv)
          out[(token * (a.nq / 2) + (kvh * GROUP + h0) / 2 + warp) * a.difference.dv + lane + 32 * k] = __float2bfloat16_rn(d[k] * f);
    }
    __syncthreads();
  }
}

// ---- host side -------------------------------------------------------------------------------

// What the two kernels of a step's shared and own positions have left, put together.
extern "C" int omnia_shared_merge_tc(const SharedAttention* given, cudaStream_t stream) {
  const SharedAttention a = *given;
  if (a.requests == 0) return 0;
  if (a.requests < 0 || a.requests > 65535 || a.nkv < 1 || a.nq != a.nkv * GROUP || a.d != D || a.dv != D || a.chunk_keys < 1 || (a.maps != 1 && a.maps != 2) ||
      (a.maps == 2 && (GROUP % 2 || a.gate || a.sink || a.difference.dv < 1 || a.difference.dv > D)) || ((uintptr_t)a.part_o & 15) || ((uintptr_t)a.part_ml & 7))
    return (int)cudaErrorInvalidValue;
  launch_pdl(shared_merge_tc_kernel, dim3(a.nkv, a.requests), 32 * MERGE_WARPS, 0, stream, a);
  return OMNIA_LAUNCH_RESULT();
}

// The pieces of all items. Pages [num_pages, 2, nkv, page_size, D], page_size a multiple of 16; q [tokens, nq, D]; an item has at most
// 2 * (128 / GROUP) * GROUP rows, its first key is a multiple of 16.
extern "C" int omnia_shared_pieces_tc(const SharedAttention* given, cudaStream_t stream) {
  const SharedAttention a = *given;
  if (a.items == 0) return 0;
  if (a.items < 0 || a.requests < 1 || a.members < 1 || a.nq != a.nkv * GROUP || a.d != D || a.dv != D || a.page_size < 16 || a.page_size % 16 ||
      a.max_pages < 1 || a.num_pages < 1 || ((uintptr_t)a.q & 15) || ((uintptr_t)a.k_pages & 15) || ((uintptr_t)a.part_o & 15) || a.softcap < 0.f ||
      (long long)a.num_pages * 2 * a.nkv * a.page_size > 0x7fffffffLL)
    return (int)cudaErrorInvalidValue;
  EncodeTiled encode = encode_tiled();
  if (encode == nullptr) return (int)cudaErrorNotSupported;
  CUtensorMap map_kv;
  const cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)a.num_pages * 2 * a.nkv * a.page_size};
  const cuuint64_t strides[1] = {(cuuint64_t)D * 2};
  const cuuint32_t box[2] = {64, 16}, elem[2] = {1, 1};
  if (encode(&map_kv, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(a.k_pages), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return (int)cudaErrorInvalidValue;
  // Queries [tokens, nq, D]: a box is the group's rows of one token, or of eight, x 64 dims.
  CUtensorMap map_q, map_q8;
  const cuuint64_t q_dims[3] = {(cuuint64_t)D, (cuuint64_t)a.nq, (cuuint64_t)a.requests};
  const cuuint64_t q_strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)a.nq * D * 2};
  cuuint32_t q_box[3] = {64, GROUP, 1};
  const cuuint32_t q_elem[3] = {1, 1, 1};
  for (int tokens = 1; tokens <= Q_MEMBERS; tokens += Q_MEMBERS - 1) {
    q_box[2] = tokens;
    if (encode(tokens == 1 ? &map_q : &map_q8, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(a.q), q_dims, q_strides, q_box, q_elem,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return (int)cudaErrorInvalidValue;
  }
  constexpr size_t smem = TILES * (size_t)TILE_BYTES + BAR_BYTES + 4 * BM * sizeof(float);
  static bool configured[64] = {};
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return (int)cudaErrorInvalidDevice;
  if (!configured[device]) {
    const cudaError_t e = cudaFuncSetAttribute(shared_pieces_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return (int)e;
    configured[device] = true;
  }
  launch_pdl(shared_pieces_tc_kernel, dim3(a.items), THREADS, smem, stream, map_kv, map_q, map_q8, a);
  return OMNIA_LAUNCH_RESULT();
}
