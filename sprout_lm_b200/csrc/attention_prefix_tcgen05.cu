// The many-row items of attention over shared prefixes on the fifth-generation tensor cores (sm_100a): whole pages that so many tokens
// share that their scores are a matrix product worth its name.
//
// A CTA owns an item of up to 256 rows, two Q tiles of 128, and walks its keys in tiles of 64:
//
//   S = Q K^T    tcgen05.mma, Q and K K-major in shared memory, S [128 x 64] in tensor memory, two buffers per Q tile
//   softmax      two warpgroups per Q tile, half a row a thread: S into registers, the halves' maxima through shared memory, P = exp2(..)
//                as bfloat16 back into tensor memory, over the first half of S's columns
//   O += P V     tcgen05.mma with P from tensor memory, V as it lies in the cache (MN-major); O stays in tensor memory
//
// as the prompt kernel of attention_maps_tcgen05.cu does, but every row sees every key, the rows are gathered from many requests, and O
// leaves unnormalised with its maximum and sum.  A row's O and sum follow its maximum only once it has grown by 2^GROWTH.  What bounds
// it: the chain S, maximum, exponentials, P, products of a tile, two tiles deep; the products alone are 1,000 cycles for 256 x 64 at head
// size 128, the exponentials 1,024, a tile takes 1,700 to 1,900.  A warp for both tiles' products took 2,300 (its waits are 150 cycles
// each, and 24 products 1,400 to issue); one warpgroup a Q tile is 3 % faster over 32,768 keys and 8 % slower over 2,000, where a CTA has
// few tiles; a quarter of the exponentials as polynomials gained 5 % there and costs 5 % here.  128 requests over 16,384 shared keys (28
// heads over 4 of 128, 30 GFLOP): 49 us, 610 TFLOP/s; the tensor pipe works 36 % of the time, the exponentials' unit 38 %.
//
// K and V come by TMA, one box per page, through a ring of stages.  Every mbarrier wait is bounded: on a timeout the CTA sets
// the status word, waits (bounded) for its copies in flight, frees its tensor memory and returns.
#include <cuda_bf16.h>

#include "attention_prefix.cuh"
#include "softmax_tmem.cuh"

using namespace sprout_prefix;

namespace {

constexpr int ROWS = 128, KEYS = 64;        // rows of a Q tile (tensor-memory lanes), keys of a tile
constexpr int THREADS = 640;                // warpgroup 0: key copies, MMA, value copies, MMA; 1, 2: softmax of Q tile 0's columns' halves; 3, 4: of Q tile 1's
constexpr int HALF = KEYS / 2;              // columns of S that a softmax thread has
constexpr int ATOM = 128 * 128;             // bytes of a [128 rows, 64 bf16] swizzled tile
constexpr int KV_ATOM = KEYS * 128;         // and of [KEYS rows, 64 bf16]
constexpr int TMEM_COLS = 512;
constexpr float GROWTH = 8.f;                // log2 of how far a row's weights may grow before its O and sum follow the maximum
constexpr int MARKS = 16;                   // tiles whose missing boxes are remembered: more than the ring's stages and the two tiles ahead

template <int DIM>
struct Layout {
  static constexpr int Q_BYTES = DIM / 64 * ATOM, KV_BYTES = DIM / 64 * KV_ATOM;
  static constexpr int STAGES = 4;
  static constexpr int OFF_K = 2 * Q_BYTES, OFF_V = OFF_K + STAGES * KV_BYTES, OFF_BAR = OFF_V + STAGES * KV_BYTES;
  static constexpr int OFF_ROWS = OFF_BAR + 512, OFF_MAX = OFF_ROWS + 2 * ROWS * 8;    // the query rows' addresses
  static constexpr int SMEM = OFF_MAX + (2 * 2 * 2 + 2) * ROWS * 4;        // the halves' maxima (two tiles), the second halves' sums
  static constexpr int O_COLUMN = 4 * KEYS;                        // tensor memory: S of the Q tiles, two buffers each, then their O
  static_assert(O_COLUMN + 2 * DIM <= TMEM_COLS, "tensor memory columns");
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

// A barrier of some of the CTA's threads, and whether all of them say so.
__device__ __forceinline__ bool named_barrier_and(int id, int threads, bool mine) {
  uint32_t all;
  asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %3, 0;\n barrier.cta.red.and.pred q, %1, %2, p;\n selp.u32 %0, 1, 0, q;\n}"
               : "=r"(all) : "r"(id), "r"(threads), "r"((uint32_t)mine) : "memory");
  return all != 0;
}
template <int DIM>
__global__ void __launch_bounds__(THREADS, 1)
attention_prefix_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Params p, const int box_rows) {
  using L = Layout<DIM>;
  constexpr int NS = L::STAGES;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sQ = smem;
  uint8_t* sK = smem + L::OFF_K;
  uint8_t* sV = smem + L::OFF_V;
  uint64_t* bars = (uint64_t*)(smem + L::OFF_BAR);
  uint64_t* k_full = bars;             // [NS] copies of a stage have landed
  uint64_t* k_empty = k_full + NS;     // the products that read a stage have completed
  uint64_t* v_full = k_empty + NS;
  uint64_t* v_empty = v_full + NS;
  uint64_t* s_full = v_empty + NS;     // [2 Q tiles][2 buffers] S is complete in tensor memory
  uint64_t* p_full = s_full + 4;       // [2][2] P is in tensor memory (8 warps arrive)
  uint64_t* o_done = p_full + 4;       // [2][2] P V of a Q tile's key tile is complete, for even and odd tiles (a waiter may be two behind)
  constexpr int BARS = 4 * NS + 12;
  uint32_t* tmem_slot = (uint32_t*)(bars + BARS);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  volatile uint32_t* missing = tmem_slot + 2;          // [MARKS] bit b: box b of the tile has no page in the pool
  static_assert(BARS * 8 + 8 + MARKS * 4 <= 512, "room for the barriers");
  static_assert(NS + 2 < MARKS, "a tile's mark outlives its reader");

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if ((smem_u32(smem) & 1023) != 0) {
    begin_items(p);
    if (tid == 0) atomicOr(p.status, SPROUT_STATUS_BAD_LAYOUT);
    end_items(p);
    return;
  }
  if (warp == 1) tmem_alloc(tmem_slot, TMEM_COLS);
  const Item item = p.items[blockIdx.x];               // whole pages: never open
  const int g = blockIdx.y, group = p.heads / p.kv_heads;
  const int* table = p.block_table + (size_t)item.table * p.table_stride;
  const bool two = item.rows > ROWS;                   // the second Q tile has rows
  const int n_tiles = (item.key_end - item.key_begin + KEYS - 1) / KEYS;

  // Q rows -> shared memory, K-major with the 128-byte swizzle (16-byte chunk c of row r at position c ^ (r & 7)); the rows' addresses first
  // (a thread that finds them one after the other, or stores a row before it asks for the next, waits for every read: 4 to 6 us in all)
  const __nv_bfloat16** from = (const __nv_bfloat16**)(smem + L::OFF_ROWS);
  if (tid < 2 * ROWS)
    from[tid] = tid < item.rows ? (const __nv_bfloat16*)p.q + (size_t)p.order[place_of_row(item, tid, group)] * p.q_stride + (size_t)head_of_row(item, tid, group, g) * DIM : nullptr;
  if (tid == THREADS - 1) {
    for (int i = 0; i < BARS; i++) {
      const bool writes_p = &bars[i] >= p_full && &bars[i] < o_done, empty = (&bars[i] >= k_empty && &bars[i] < v_full) || (&bars[i] >= v_empty && &bars[i] < s_full);
      mbar_init(&bars[i], writes_p ? 8 : empty && two ? 2 : 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  begin_items(p);
  __syncthreads();
  int issued = 0;                                     // tiles whose copies were issued (copy warps)
  auto gave_up = [&]() { *abort_flag = 1; atomicOr(p.status, SPROUT_STATUS_WAIT_TIMEOUT); };
  if (warp != 0 && warp != 2) {                        // the copies start meanwhile
    const int other = tid - (warp == 1 ? 32 : 64);
    constexpr int CHUNKS = DIM / 8, OTHERS = THREADS - 64, EACH = (2 * ROWS * CHUNKS + OTHERS - 1) / OTHERS;
    uint4 held[EACH];                                    // all on their way before the first is stored
  #pragma unroll
    for (int k = 0; k < EACH; k++) {
      const int idx = other + k * OTHERS, i = min(idx / CHUNKS, 2 * ROWS - 1);
      const __nv_bfloat16* at = from[i];
      held[k] = at != nullptr ? *(const uint4*)(at + idx % CHUNKS * 8) : make_uint4(0, 0, 0, 0);
    }
  #pragma unroll
    for (int k = 0; k < EACH; k++) {
      const int idx = other + k * OTHERS, i = idx / CHUNKS, c = idx % CHUNKS, q = i >> 7, row = i & (ROWS - 1);
      if (i < 2 * ROWS) *(uint4*)(sQ + q * L::Q_BYTES + (c >> 3) * ATOM + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = held[k];
    }
    fence_proxy_async();
    tc_fence_before();
    named_barrier(1, OTHERS);
    tc_fence_after();
  }
  const uint32_t tmem_base = *tmem_slot;
  if (warp < 4) {
    // the launch's 640 x 96 registers as 128 x 64 and 512 x 104
    warpgroup_regs_give<64>();
    if (warp == 0 || warp == 2) {
      // ---------------- copies, keys by warp 0 and values by warp 2: one TMA box per page (or per KEYS keys of a larger page); lane b
      // issues box b's copies, lane 0 waits for the stage and posts the bytes.  The page of a tile is looked up while the tile before
      // waits and is copied.
      const bool keys = warp == 0;
      const CUtensorMap* map = keys ? &map_k : &map_v;
      uint64_t* full = keys ? k_full : v_full;
      uint64_t* empty = keys ? k_empty : v_empty;
      const uint32_t stages = smem_u32(keys ? sK : sV);
      const int boxes = KEYS / box_rows;
      auto box_key = [&](int j) {                     // the first key of this lane's box of tile j, -1 beyond the range
        const int key = item.key_begin + j * KEYS + lane * box_rows;
        return lane >= boxes || key >= item.key_end ? -1 : key;
      };
      int key = box_key(0);
      int page = key >= 0 ? table[key / p.page_tokens] : 0;
      for (int j = 0; j < n_tiles; j++) {
        const int s = j % NS;
        const bool bad = key >= 0 && (page < 0 || page >= p.num_pages);
        if (bad) atomicOr(p.status, SPROUT_STATUS_BAD_PAGE);
        const unsigned marks = __ballot_sync(0xffffffffu, bad);
        const int row_at = key < 0 || bad ? -1 : (page * p.kv_heads + g) * p.page_tokens + key % p.page_tokens;
        if (j + 1 < n_tiles) {
          key = box_key(j + 1);
          if (key >= 0) page = table[key / p.page_tokens];
        }
        const uint32_t bytes = (uint32_t)__popc(__ballot_sync(0xffffffffu, row_at >= 0)) * box_rows * DIM * 2;
        bool ok = true;
        if (lane == 0) {
          ok = !*abort_flag && mbar_wait(&empty[s], ((j / NS) & 1) ^ 1, abort_flag);
          if (keys) missing[j % MARKS] = marks;
          if (ok) mbar_expect_tx(&full[s], bytes);
          else gave_up();
        }
        if (!__shfl_sync(0xffffffffu, ok, 0)) break;
        if (row_at >= 0)
          for (int a = 0; a < DIM / 64; a++)
            tma_load_2d_addr(stages + s * L::KV_BYTES + a * KV_ATOM + lane * box_rows * 128, map, smem_u32(&full[s]), a * 64, row_at);
        issued = j + 1;
      }
    } else if (warp == 1 || two) {
      // ---------------- MMA issuers, warp 1 for the first Q tile and warp 3 for the second: S(0) and S(1), then for every key tile
      // [P(j)] P V(j), S(j + 2).  (One warp for both took 2,300 cycles a tile, 1,400 of them to issue 24 products and the rest in waits
      // that found what they waited for.)  The products that read a stage release it.  The whole warp walks the loop on values that are
      // the same in all lanes (they stay in uniform registers, where the products take them from); one elected lane issues.
      const int q = __shfl_sync(0xffffffffu, warp >> 1, 0);
      const uint32_t idesc_s = umma_idesc(ROWS, KEYS), idesc_o = umma_idesc_b_mn(ROWS, DIM);
      const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base, 0);
      const int tiles = __shfl_sync(0xffffffffu, n_tiles, 0);
      const uint32_t k0 = (smem_u32(sK) & 0x3FFFF) >> 4, v0 = (smem_u32(sV) & 0x3FFFF) >> 4, q0 = ((smem_u32(sQ) & 0x3FFFF) + q * L::Q_BYTES) >> 4;
      const uint32_t bar0 = smem_u32(bars);
      auto bar_of = [&](const uint64_t* bar) { return bar0 + (uint32_t)((const char*)bar - (const char*)bars); };
      auto wait = [&](uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait_addr(bar, parity, abort_flag)) != 0; };
      // descriptors: the start address / 16 in the low word, layout constants (umma_smem_desc, umma_smem_desc_mn) in the high one
      constexpr uint32_t DESC_HI = (1024 >> 4) | (1u << 14) | (2u << 29);
      auto issue_s = [&](int stage, int buf) {
        if (elect_one()) {
#pragma unroll
          for (int a = 0; a < DIM / 64; a++)
#pragma unroll
            for (int kk = 0; kk < 4; kk++)
              umma_bf16_words(tmem + (q * 2 + buf) * KEYS, q0 + a * (ATOM / 16) + 2 * kk, DESC_HI,
                              k0 + stage * (L::KV_BYTES / 16) + a * (KV_ATOM / 16) + 2 * kk, DESC_HI, idesc_s, (a | kk) != 0);
          umma_commit_addr(bar_of(s_full) + (q * 2 + buf) * 8);
          umma_commit_addr(bar_of(k_empty) + stage * 8);
        }
        __syncwarp();
      };
      auto issue_pv = [&](int stage, int buf, bool first) {
        if (elect_one()) {
#pragma unroll
          for (int ks = 0; ks < KEYS / 16; ks++)
            umma_bf16_from_tmem_words(tmem + L::O_COLUMN + q * DIM, tmem + (q * 2 + buf) * KEYS + ks * 8,
                                      (v0 + stage * (L::KV_BYTES / 16) + ks * 128) | ((uint32_t)(KV_ATOM >> 4) << 16), DESC_HI, idesc_o, !first || ks != 0);
          umma_commit_addr(bar_of(o_done) + (q * 2 + buf) * 8);
          umma_commit_addr(bar_of(v_empty) + stage * 8);
        }
        __syncwarp();
      };
      bool ok = true;
      int k_stage = 0, v_stage = 0;                    // running stages and parities of the rings
      uint32_t k_parity = 0, v_parity = 0;
      for (int j = 0; j < min(2, tiles) && ok; j++) {
        ok = wait(bar_of(k_full) + k_stage * 8, 0);
        if (!ok) break;
        tc_fence_after();
        issue_s(k_stage, j);
        k_stage++;
      }
      for (int j = 0; j < tiles && ok; j++) {
        const int buf = j & 1;
        const uint32_t parity = (j >> 1) & 1;
        ok = wait(bar_of(v_full) + v_stage * 8, v_parity);
        if (ok && j + 2 < tiles) ok = wait(bar_of(k_full) + k_stage * 8, k_parity);
        if (!ok) break;
        ok = wait(bar_of(p_full) + (q * 2 + buf) * 8, parity);
        if (!ok) break;
        tc_fence_after();
        issue_pv(v_stage, buf, j == 0);
        if (j + 2 < tiles) issue_s(k_stage, buf);
        if (++k_stage == NS) { k_stage = 0; k_parity ^= 1; }
        if (++v_stage == NS) { v_stage = 0; v_parity ^= 1; }
      }
      if (!ok && lane == 0) gave_up();
    }
  } else {
    // ---------------- softmax: two warpgroups per Q tile, half a row a thread
    warpgroup_regs_take<104>();
    const int q = ((warp >> 2) - 1) >> 1, half = ((warp >> 2) - 1) & 1, quarter = warp & 3, row = quarter * 32 + lane;       // a warp reads tensor-memory lanes 32 * (warp % 4) on
    const int i = q * ROWS + row;                      // of the item
    const int my_tiles = q == 0 || two ? n_tiles : 0;
    const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const uint32_t o_addr = lane_addr + L::O_COLUMN + q * DIM;
    const float scale_log2 = p.scale_log2;
    const uint64_t scale2 = pair(scale_log2, scale_log2);
    float* maxima = (float*)(smem + L::OFF_MAX) + q * 2 * ROWS + row;        // [2 tiles][2 Q tiles][2 halves][128]
    float* second = (float*)(smem + L::OFF_MAX) + 8 * ROWS + q * ROWS + row; // [2 Q tiles][128]
    const int meet = 2 + q * 4 + quarter;              // the barrier of the two warps that share 32 rows
    float m = -INFINITY;                               // the maximum that the sums stand for (unscaled scores)
    uint64_t l2 = 0ull;                                // the sum, as two partial sums
    bool ok = true;
    for (int j = 0; j < my_tiles; j++) {
      const uint32_t s_addr = lane_addr + (q * 2 + (j & 1)) * KEYS;
      ok = !*abort_flag && mbar_wait(&s_full[q * 2 + (j & 1)], (j >> 1) & 1, abort_flag);
      if (!ok) gave_up();
      ok = __all_sync(0xffffffffu, ok);                // one that gave up goes on to where it meets the other half
      tc_fence_after();
      uint32_t sc[HALF];
      tmem_load32_issue(s_addr + half * HALF, sc);
      tmem_load_wait(sc);
      const int there = item.key_end - item.key_begin - j * KEYS - half * HALF;        // of this half's keys before the range's end
      const uint32_t marks = missing[j % MARKS];
      if (there < HALF || marks != 0) {
#pragma unroll
        for (int k = 0; k < HALF; k++) if (k >= there || (marks >> ((half * HALF + k) / box_rows) & 1)) sc[k] = 0xff800000u;          // -inf
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int k = 0; k < HALF; k += 2) mx[(k >> 1) & 3] = max3(mx[(k >> 1) & 3], __uint_as_float(sc[k]), __uint_as_float(sc[k + 1]));
      float n = max3(max3(m, mx[0], mx[1]), mx[2], mx[3]);
      float* at = maxima + (j & 1) * 4 * ROWS;
      at[half * ROWS] = n;
      ok = named_barrier_and(meet, 64, ok);            // both halves are in registers: P may go over S
      if (!ok) break;
      n = max3(n, at[(half ^ 1) * ROWS], n);
      // it moved: bring O and the sum to it (by less than 2^GROWTH: they stay, and weights are up to that large)
      const bool moved = m == -INFINITY ? n != m : (n - m) * scale_log2 > GROWTH;
      if (__any_sync(0xffffffffu, moved)) {
        const float alpha = !moved ? 1.0f : m == -INFINITY ? 0.f : exp2_fast((m - n) * scale_log2);
        if (moved) m = n;
        float lo2, hi2;
        unpair(l2, lo2, hi2);
        l2 = pair(lo2 * alpha, hi2 * alpha);
        if (j > 0) {
          // a timeout here shows in the status word and the abort flag; the halves go on in step, to the next wait for S
          if (*abort_flag || !mbar_wait(&o_done[q * 2 + ((j - 1) & 1)], ((j - 1) >> 1) & 1, abort_flag)) gave_up();
          __syncwarp();
          tc_fence_after();
          for (int c = half * (DIM / 2); c < (half + 1) * (DIM / 2); c += 16) {
            uint32_t o[16];
            tmem_load16(o_addr + c, o);
#pragma unroll
            for (int k = 0; k < 16; k++) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
            tmem_store16(o_addr + c, o);
          }
        }
      }
      const float base = m == -INFINITY ? 0.f : m * scale_log2;
      const uint64_t nbase2 = pair(-base, -base);
      // probabilities, their sum, and P as bfloat16 into tensor memory
      uint64_t sums[2] = {0ull, 0ull};
      uint32_t packed[HALF / 2];
#pragma unroll
      for (int k = 0; k < HALF; k += 2) {
        float x0, x1;
        unpair(fma2(pair(sc[k], sc[k + 1]), scale2, nbase2), x0, x1);
        const float p0 = exp2_fast(x0), p1 = exp2_fast(x1);
        __nv_bfloat162 h = __floats2bfloat162_rn(p0, p1);
        packed[k >> 1] = *(uint32_t*)&h;
        sums[(k >> 1) & 1] = add2(sums[(k >> 1) & 1], pair(p0, p1));
      }
      tmem_store16(s_addr + half * (HALF / 2), packed);
      l2 = add2(l2, add2(sums[0], sums[1]));
      tmem_store_wait();
      // V rows that no copy filled (behind the range's end, or of a page outside the pool) hold what lay there before, an infinity or a NaN
      // of the ring's tile before among it: their probabilities are zero, but zero times those is not.  They are cleared once the copies
      // have landed, by each Q tile before it signals its P; four threads a row.
      if (there + half * HALF < KEYS || marks != 0) {
        const int s = j % NS, key = row & (KEYS - 1), share = half * 2 + (row >> 6);
        if (*abort_flag || !mbar_wait(&v_full[s], (j / NS) & 1, abort_flag)) gave_up();
        if (key >= there + half * HALF || (marks >> (key / box_rows) & 1)) {
#pragma unroll
          for (int k = 0; k < DIM / 32; k++) {
            const int c = share * (DIM / 32) + k;
            *(uint4*)(sV + s * L::KV_BYTES + (c >> 3) * KV_ATOM + key * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
        }
        fence_proxy_async();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[q * 2 + (j & 1)]);
    }
    if (ok && my_tiles > 0) {
      ok = !*abort_flag && mbar_wait(&o_done[q * 2 + ((my_tiles - 1) & 1)], ((my_tiles - 1) >> 1) & 1, abort_flag);
      if (!ok) gave_up();
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
    }
    if (my_tiles > 0) {
      // O leaves by way of the Q tile's room, which no product reads any more: a warp's 32 rows, COLUMNS columns at a time, so that its
      // stores are whole lines
      constexpr int COLUMNS = DIM / 4, CHUNKS16 = COLUMNS / 4, AT_ONCE = 32 / CHUNKS16;        // 16-byte chunks of a row, rows a store
      float l_lo, l_hi;
      unpair(l2, l_lo, l_hi);
      if (half == 1) *second = l_lo + l_hi;
      ok = named_barrier_and(meet, 64, ok);            // both halves have their outputs, or both leave
      size_t slot = 0;
      const bool mine = ok && i < item.rows;
      if (mine) {
        slot = (size_t)(p.part_start[place_of_row(item, i, group)] + item.part) * p.heads + head_of_row(item, i, group, g);
        if (half == 0) p.part_sum[slot] = make_float2(m == -INFINITY ? -INFINITY : m * scale_log2, l_lo + l_hi + *second);
      }
      const unsigned long long to = mine ? (unsigned long long)(p.part_out + slot * DIM) : 0ull;
      float* dst[CHUNKS16];                            // of the rows that this lane stores a chunk of
#pragma unroll
      for (int k = 0; k < CHUNKS16; k++) dst[k] = (float*)__shfl_sync(0xffffffffu, to, k * AT_ONCE + lane / CHUNKS16);
      float* room = (float*)(sQ + q * L::Q_BYTES) + (half * 4 + quarter) * (32 * COLUMNS);       // chunk c of row r at c ^ (r & (CHUNKS16 - 1))
      for (int c = half * (DIM / 2); c < (half + 1) * (DIM / 2); c += COLUMNS) {
        uint32_t o[COLUMNS];
        if constexpr (COLUMNS == 32) tmem_load32(o_addr + c, o);
        else tmem_load16(o_addr + c, o);
        __syncwarp();
#pragma unroll
        for (int k = 0; k < CHUNKS16; k++) *(uint4*)(room + lane * COLUMNS + ((k ^ (lane & (CHUNKS16 - 1))) << 2)) = make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
        __syncwarp();
#pragma unroll
        for (int k = 0; k < CHUNKS16; k++) {
          const int r = k * AT_ONCE + lane / CHUNKS16, chunk = lane % CHUNKS16;
          if (dst[k] != nullptr) *(uint4*)(dst[k] + c + chunk * 4) = *(const uint4*)(room + r * COLUMNS + ((chunk ^ (r & (CHUNKS16 - 1))) << 2));
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag && (warp == 0 || warp == 2) && lane == 0) {
    // copies already issued still write shared memory: wait for them (bounded) before leaving
    uint64_t* full = warp == 0 ? k_full : v_full;
    for (int j = max(0, issued - NS); j < issued; j++) mbar_wait(&full[j % NS], (j / NS) & 1);
  }
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem_base, TMEM_COLS);
  end_items(p);
}

template <int DIM>
int launch(const CUtensorMap& map_k, const CUtensorMap& map_v, const Params& p, int items, int box_rows, cudaStream_t stream) {
  using L = Layout<DIM>;
  if (reserve_shared<attention_prefix_tc_kernel<DIM>>(L::SMEM, "attention_shared_prefix (tcgen05)")) return 1;
  sprout_launch(attention_prefix_tc_kernel<DIM>, dim3(items, p.kv_heads), dim3(THREADS), L::SMEM, stream, map_k, map_v, p, box_rows);
  return sprout_check_launch("attention_shared_prefix (tcgen05)");
}

}  // namespace

// Whether segments of whole pages may run here: the cache's sizes and its rows' number as a tensor map's coordinate.
SPROUT_API int sprout_attention_prefix_tc_supported(int head_dim, int page_tokens) {
  return (head_dim == 64 || head_dim == 128) && (page_tokens == 8 || page_tokens == 16 || page_tokens == 32 || page_tokens == 64 || (page_tokens > 0 && page_tokens % 128 == 0));
}

int sprout_attention_prefix_tc(const Params& p, int items, cudaStream_t stream) {
  SPROUT_REQUIRE(sprout_attention_prefix_tc_supported(p.head_dim, p.page_tokens), "attention_shared_prefix (tcgen05): head_dim %d or page size %d is not taken", p.head_dim, p.page_tokens);
  const long long cache_rows = (long long)p.num_pages * p.kv_heads * p.page_tokens;
  SPROUT_REQUIRE(cache_rows <= 0x7fffffffLL, "attention_shared_prefix (tcgen05): the cache has too many rows for a tensor map coordinate");
  const int box_rows = p.page_tokens < KEYS ? p.page_tokens : KEYS;
  CUtensorMap map_k, map_v;
  if (tensor_map(p.k_cache, (int)cache_rows, p.head_dim, p.head_dim, box_rows, &map_k)) return 1;
  if (tensor_map(p.v_cache, (int)cache_rows, p.head_dim, p.head_dim, box_rows, &map_v)) return 1;
  return p.head_dim == 64 ? launch<64>(map_k, map_v, p, items, box_rows, stream) : launch<128>(map_k, map_v, p, items, box_rows, stream);
}
