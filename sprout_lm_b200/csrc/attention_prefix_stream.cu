// The few-row items of attention over shared prefixes: streams of keys and values, bfloat16, head sizes 64 and 128, pages that TMA copies a
// box at a time (attention_prefix.cu has a kernel for all others).
//
// A CTA walks (item, key/value head) pairs in steps of 64 keys.  One warp copies: a box per page and 64 columns, through a ring of stages,
// over the ends of pairs.  Four warps compute, the item's up to 16 rows one tile of mma.sync: of a step's scores a warp has 16 keys; the
// warps agree on the maxima through shared memory, put their weights there side by side, and each multiplies all of them with its share
// of the columns, so that outputs need no merging.  The query rows of a pair are read while the pair before is computed.
//
// What bounds it is memory where the items are many, up to the walk's end, where the last pairs of some CTAs run alone: 128 requests of 1,500
// keys of their own (28 heads over 4 of 128) 395 MB in 76 us, 5.2 TB/s, cold.  What is in flight does not: head size 128 has room for two
// CTAs an SM, each with up to 96 KB on its way, and 44 KB an SM cover a microsecond at the full rate.  A short walk is bound by a step's
// chain: scores, maximum, barrier, exponentials, barrier, products, 1.1 us.  With the copies issued by the computing warps (cp.async, some
// twelve instructions a thread and 16 bytes) their instructions bounded it: 4.9 TB/s at three CTAs an SM, 3.7 with a ring of three stages
// at two.
//
// Every mbarrier wait is bounded: on a timeout the CTA sets the status word, waits (bounded) for its copies in flight and returns.
#include "attention_bf16.cuh"
#include "attention_prefix.cuh"
#include "tcgen05.cuh"

using namespace sprout_prefix;
using namespace sprout_attn;

namespace {

constexpr int KEYS = 64, THREADS = 160, COMPUTE = 128;         // keys of a step; four computing warps and one that copies
constexpr int ATOM = KEYS * 128;                               // bytes of [KEYS rows, 64 bf16]

template <int HD>
struct Layout {
  static constexpr int STAGES = HD == 128 ? 3 : 4, CTAS = HD == 128 ? 2 : 3;         // CTAs an SM
  static constexpr int KV_BYTES = HD / 64 * ATOM, STAGE_BYTES = 2 * KV_BYTES;        // keys, then values
  static constexpr int Q_STRIDE = HD + 8, P_STRIDE = KEYS + 8;
  static constexpr int OFF_Q = STAGES * STAGE_BYTES, OFF_P = OFF_Q + 16 * Q_STRIDE * 2, OFF_F = OFF_P + 16 * P_STRIDE * 2, OFF_BAR = OFF_F + 2 * 64 * 4;
  static constexpr int SMEM = OFF_BAR + 128;
};

__device__ __forceinline__ void compute_barrier() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
// The same; whether all threads say so.
__device__ __forceinline__ bool compute_barrier_and(bool mine) {
  uint32_t all;
  asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n barrier.cta.red.and.pred q, 1, 128, p;\n selp.u32 %0, 1, 0, q;\n}" : "=r"(all) : "r"((uint32_t)mine) : "memory");
  return all != 0;
}

// LATER: the plan serves later steps too (Params::stretch).  Looking whether an item is open costs 0.3 to 0.9 us a launch: few items 7.0 us
// without and 7.4 with, a long walk 47.0 and 47.9.
template <int HD, bool LATER>
__global__ void __launch_bounds__(THREADS, Layout<HD>::CTAS)
attention_prefix_stream_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Params p, const int pairs, const int box_rows) {
  using L = Layout<HD>;
  constexpr int NS = L::STAGES, PIECES = HD / 8, MINE = HD / 64;       // MINE: a warp's groups of 16 columns
  extern __shared__ __align__(1024) uint8_t smem[];
  __nv_bfloat16* sQ = (__nv_bfloat16*)(smem + L::OFF_Q);               // [16][Q_STRIDE]
  __nv_bfloat16* sP = (__nv_bfloat16*)(smem + L::OFF_P);               // [16][P_STRIDE]
  float* s_max = (float*)(smem + L::OFF_F);                            // [4 warps][16]
  float* s_sum = s_max + 64;                                           // [4][16]
  uint64_t* full = (uint64_t*)(smem + L::OFF_BAR);                     // [NS] copies of a stage have landed
  uint64_t* empty = full + NS;                                         // [NS] the four warps are done with it
  volatile uint32_t* missing = (uint32_t*)(empty + NS);                // [NS] bit b: box b of the stage has no page in the pool
  volatile uint32_t* abort_flag = missing + NS;
  static_assert(NS * 20 + 4 <= 128, "room for the barriers");
  const int group = p.heads / p.kv_heads, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if ((smem_u32(smem) & 1023) != 0) {
    begin_items(p);
    if (tid == 0) atomicOr(p.status, SPROUT_STATUS_BAD_LAYOUT);
    end_items(p);
    return;
  }
  if (tid == 0) {
    for (int i = 0; i < NS; i++) { mbar_init(&full[i], 1); mbar_init(&empty[i], 4); }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // pairs come longest first; a CTA takes one of every round, forwards and backwards in turn
  auto pair_of = [&](int round) {
    const long long index = (long long)round * gridDim.x + (round & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
    return index < pairs ? (int)index : -1;
  };
  int pair = pair_of(0), next_pair = pair_of(1);       // the grid has at most as many CTAs as there are pairs
  Item item = p.items[pair / p.kv_heads], next_item = p.items[max(next_pair, 0) / p.kv_heads];
  begin_items(p);
  if (LATER) {
    item = in_step(p, item);
    next_item = in_step(p, next_item);
  }
  __syncthreads();
  auto item_of = [&](int pair) {
    const Item planned = p.items[max(pair, 0) / p.kv_heads];
    return LATER ? in_step(p, planned) : planned;
  };
  auto gave_up = [&]() { *abort_flag = 1; atomicOr(p.status, SPROUT_STATUS_WAIT_TIMEOUT); };
  int steps = 0;                                       // whose copies were issued (the copying warp), or that were computed
  if (warp == 4) {
    // lane b copies box b of a step, keys and values; lane 0 waits for the stage and posts the bytes.  The page of a step is looked up while
    // the step before waits and is copied.
    const uint32_t stages = smem_u32(smem);
    asm volatile("fence.proxy.async.global;" ::: "memory");        // the gate told ordinary accesses of the cache's writes, the copies go another way
    const int boxes = KEYS / box_rows;
    int round = 0;
    int base = item.key_begin;
    auto box_key = [&]() {
      const int key = base + lane * box_rows;
      return lane < boxes && pair >= 0 && key < item.key_end ? key : -1;
    };
    auto page_of = [&](int key) { return key >= 0 ? p.block_table[(size_t)item.table * p.table_stride + key / p.page_tokens] : 0; };
    int key = box_key(), page = page_of(key);
    while (pair >= 0) {
      const int s = steps % NS, g = pair % p.kv_heads;
      const bool bad = key >= 0 && (page < 0 || page >= p.num_pages);
      if (bad) atomicOr(p.status, SPROUT_STATUS_BAD_PAGE);
      const unsigned marks = __ballot_sync(0xffffffffu, bad);
      const int row = key < 0 || bad ? -1 : (page * p.kv_heads + g) * p.page_tokens + key % p.page_tokens;
      base += KEYS;
      if (base >= item.key_end) {
        round++;
        pair = next_pair;
        item = next_item;
        base = item.key_begin;
        next_pair = pair_of(round + 1);
        next_item = item_of(next_pair);
      }
      key = box_key();
      page = page_of(key);
      const uint32_t bytes = (uint32_t)__popc(__ballot_sync(0xffffffffu, row >= 0)) * box_rows * HD * 4;
      bool ok = true;
      if (lane == 0) {
        ok = !*abort_flag && mbar_wait(&empty[s], ((steps / NS) & 1) ^ 1, abort_flag);
        missing[s] = marks;
        if (ok) mbar_expect_tx(&full[s], bytes);
        else gave_up();
      }
      if (!__shfl_sync(0xffffffffu, ok, 0)) break;
      if (row >= 0) {
        const uint32_t to = stages + s * L::STAGE_BYTES + lane * box_rows * 128;
#pragma unroll
        for (int a = 0; a < HD / 64; a++) {
          tma_load_2d_addr(to + a * ATOM, &map_k, smem_u32(&full[s]), a * 64, row);
          tma_load_2d_addr(to + L::KV_BYTES + a * ATOM, &map_v, smem_u32(&full[s]), a * 64, row);
        }
      }
      steps++;
    }
    __syncwarp();
    if (*abort_flag && lane == 0)                      // copies already issued still write shared memory: wait for them (bounded) before leaving
      for (int j = max(0, steps - NS); j < steps; j++) mbar_wait(&full[j % NS], (j / NS) & 1);
    __syncwarp();
    end_items(p);
    return;
  }

  const int gr = lane >> 2, qc = lane & 3;
  // element (row, 16-byte piece) of a swizzled [KEYS, HD] tile
  auto at = [](const uint8_t* tile, int row, int piece) { return tile + (piece >> 3) * ATOM + row * 128 + (((piece & 7) ^ (row & 7)) << 4); };
  constexpr int EACH = 16 * PIECES / COMPUTE;
  auto query = [&](const Item& item, int g, uint4 (&q)[EACH]) {
#pragma unroll
    for (int k = 0; k < EACH; k++) {
      const int idx = tid + k * COMPUTE, i = idx / PIECES;
      q[k] = make_uint4(0, 0, 0, 0);
      if (i < item.rows)
        q[k] = *(const uint4*)((const __nv_bfloat16*)p.q + (size_t)p.order[place_of_row(item, i, group)] * p.q_stride + (size_t)head_of_row(item, i, group, g) * HD + idx % PIECES * 8);
    }
  };
  uint4 q[EACH];
  query(item, pair % p.kv_heads, q);
  bool ok = true;
  for (int round = 0; pair >= 0; round++) {
    const int g = pair % p.kv_heads;
    size_t slot[2];
#pragma unroll
    for (int half = 0; half < 2; half++) {
      const int i = min(gr + half * 8, item.rows - 1);
      slot[half] = (size_t)(p.part_start[place_of_row(item, i, group)] + item.part) * p.heads + head_of_row(item, i, group, g);
    }
    // the tile's rows of the pair before were last read before its last barrier
#pragma unroll
    for (int k = 0; k < EACH; k++) { const int idx = tid + k * COMPUTE; *(uint4*)(sQ + idx / PIECES * L::Q_STRIDE + idx % PIECES * 8) = q[k]; }
    compute_barrier();
    if (round > 0) {
      next_pair = pair_of(round + 1);
      next_item = item_of(next_pair);
    }
    if (next_pair >= 0) query(next_item, next_pair % p.kv_heads, q);
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f, o[2 * MINE][4];
#pragma unroll
    for (int n = 0; n < 2 * MINE; n++) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    for (int base = item.key_begin; base < item.key_end; base += KEYS) {
      const int stage = steps % NS, there = item.key_end - base;       // keys of the step before the range's end, KEYS and more: all
      uint8_t* k = smem + stage * L::STAGE_BYTES;
      uint8_t* v = k + L::KV_BYTES;
      ok = !*abort_flag && mbar_wait(&full[stage], (steps / NS) & 1, abort_flag);
      if (!ok) gave_up();
      const uint32_t marks = missing[stage];
      const bool holes = there < KEYS || marks != 0;
      if (holes) {
        // what no copy filled, or what a page holds behind the range: finite (its weight is zero, and zero times a NaN is not)
        for (int idx = tid; idx < KEYS * PIECES; idx += COMPUTE) {
          const int row = idx / PIECES;
          if (row >= there || (marks >> (row / box_rows) & 1)) *(uint4*)at(v, row, idx % PIECES) = make_uint4(0, 0, 0, 0);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      float s[2][4];
#pragma unroll
      for (int n = 0; n < 2; n++) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
      for (int kk = 0; kk < HD / 16; kk++) {
        uint32_t a[4], b[4];                           // b: 16 keys, fragments of two MMAs
        ldmatrix_x4(a, sQ + (lane & 15) * L::Q_STRIDE + kk * 16 + (lane >> 4) * 8);
        ldmatrix_x4(b, at(k, warp * 16 + (lane & 7) + ((lane >> 4) << 3), kk * 2 + ((lane >> 3) & 1)));
        mma_bf16(s[0], a, b[0], b[1]);
        mma_bf16(s[1], a, b[2], b[3]);
      }
      float top0 = -INFINITY, top1 = -INFINITY;
#pragma unroll
      for (int n = 0; n < 2; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) s[n][i] *= p.scale_log2;
      if (holes)
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
          for (int i = 0; i < 2; i++) {
            const int row = warp * 16 + n * 8 + qc * 2 + i;
            if (row >= there || (marks >> (row / box_rows) & 1)) s[n][i] = s[n][2 + i] = -INFINITY;
          }
#pragma unroll
      for (int n = 0; n < 2; n++) {
        top0 = fmaxf(top0, fmaxf(s[n][0], s[n][1]));
        top1 = fmaxf(top1, fmaxf(s[n][2], s[n][3]));
      }
      top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, 1));
      top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, 2));
      top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, 1));
      top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, 2));
      if (qc == 0) { s_max[warp * 16 + gr] = top0; s_max[warp * 16 + gr + 8] = top1; }
      ok = compute_barrier_and(ok);                    // the maxima are there, and all are done with the weights of the step before
      if (!ok) break;
      top0 = m0;
      top1 = m1;
#pragma unroll
      for (int w = 0; w < 4; w++) { top0 = fmaxf(top0, s_max[w * 16 + gr]); top1 = fmaxf(top1, s_max[w * 16 + gr + 8]); }
      const float alpha0 = m0 == -INFINITY ? 0.f : exp2_fast(m0 - top0), alpha1 = m1 == -INFINITY ? 0.f : exp2_fast(m1 - top1);
      m0 = top0;
      m1 = top1;
      const float base0 = m0 == -INFINITY ? 0.f : m0, base1 = m1 == -INFINITY ? 0.f : m1;
      l0 *= alpha0;
      l1 *= alpha1;
#pragma unroll
      for (int n = 0; n < 2; n++) {
        const float e0 = exp2_fast(s[n][0] - base0), e1 = exp2_fast(s[n][1] - base0), e2 = exp2_fast(s[n][2] - base1), e3 = exp2_fast(s[n][3] - base1);
        l0 += e0 + e1;
        l1 += e2 + e3;
        *(uint32_t*)(sP + gr * L::P_STRIDE + warp * 16 + n * 8 + qc * 2) = pack_bf16(e0, e1);
        *(uint32_t*)(sP + (gr + 8) * L::P_STRIDE + warp * 16 + n * 8 + qc * 2) = pack_bf16(e2, e3);
      }
#pragma unroll
      for (int n = 0; n < 2 * MINE; n++) { o[n][0] *= alpha0; o[n][1] *= alpha0; o[n][2] *= alpha1; o[n][3] *= alpha1; }
      if (base + KEYS >= item.key_end) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
        l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
        if (qc == 0) { s_sum[warp * 16 + gr] = l0; s_sum[warp * 16 + gr + 8] = l1; }
      }
      compute_barrier();                               // the weights are there
#pragma unroll
      for (int j = 0; j < KEYS / 16; j++) {
        uint32_t a[4];
        ldmatrix_x4(a, sP + (lane & 15) * L::P_STRIDE + j * 16 + (lane >> 4) * 8);
#pragma unroll
        for (int n = 0; n < MINE; n++) {
          uint32_t b[4];
          ldmatrix_x4_trans(b, at(v, j * 16 + (lane & 15), (warp * MINE + n) * 2 + (lane >> 4)));
          mma_bf16(o[2 * n], a, b[0], b[1]);
          mma_bf16(o[2 * n + 1], a, b[2], b[3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[stage]);
      steps++;
    }
    if (!ok) break;
#pragma unroll
    for (int half = 0; half < 2; half++) {
      const int i = gr + half * 8;
      if (i >= item.rows) continue;
#pragma unroll
      for (int n = 0; n < MINE; n++) {
        float* to = p.part_out + slot[half] * HD + (warp * MINE + n) * 16 + qc * 2;
        *(float2*)to = make_float2(o[2 * n][half * 2], o[2 * n][half * 2 + 1]);
        *(float2*)(to + 8) = make_float2(o[2 * n + 1][half * 2], o[2 * n + 1][half * 2 + 1]);
      }
      if (warp == 0 && qc == 0) p.part_sum[slot[half]] = make_float2(half ? m1 : m0, s_sum[i] + s_sum[16 + i] + s_sum[32 + i] + s_sum[48 + i]);
    }
    pair = next_pair;
    item = next_item;
  }
  end_items(p);
}

template <int HD, bool LATER>
int launch(const CUtensorMap& map_k, const CUtensorMap& map_v, const Params& p, int items, int ctas, int box_rows, cudaStream_t stream) {
  using L = Layout<HD>;
  if (reserve_shared<attention_prefix_stream_kernel<HD, LATER>>(L::SMEM, "attention_shared_prefix (few rows)")) return 1;
  const long long pairs = (long long)items * p.kv_heads, most = (long long)L::CTAS * sprout_sm_count(), slots = ctas < most ? ctas : most;
  SPROUT_REQUIRE(pairs <= 0x7fffffffLL, "attention_shared_prefix: too many items");
  sprout_launch(attention_prefix_stream_kernel<HD, LATER>, dim3((unsigned)(pairs < slots ? pairs : slots)), dim3(THREADS), L::SMEM, stream, map_k, map_v, p, (int)pairs, box_rows);
  return sprout_check_launch("attention_shared_prefix (few rows)");
}

}  // namespace

// Items of up to 16 rows; the sizes are sprout_attention_prefix_tc_supported's.
int sprout_attention_prefix_stream(const Params& p, int items, int ctas, cudaStream_t stream) {
  const long long cache_rows = (long long)p.num_pages * p.kv_heads * p.page_tokens;
  SPROUT_REQUIRE(cache_rows <= 0x7fffffffLL && (p.head_dim == 64 || p.head_dim == 128), "attention_shared_prefix (few rows): sizes that are not taken");
  const int box_rows = p.page_tokens < KEYS ? p.page_tokens : KEYS;
  CUtensorMap map_k, map_v;
  if (tensor_map(p.k_cache, (int)cache_rows, p.head_dim, p.head_dim, box_rows, &map_k)) return 1;
  if (tensor_map(p.v_cache, (int)cache_rows, p.head_dim, p.head_dim, box_rows, &map_v)) return 1;
  if (p.head_dim == 64) return p.stretch > 0 ? launch<64, true>(map_k, map_v, p, items, ctas, box_rows, stream) : launch<64, false>(map_k, map_v, p, items, ctas, box_rows, stream);
  return p.stretch > 0 ? launch<128, true>(map_k, map_v, p, items, ctas, box_rows, stream) : launch<128, false>(map_k, map_v, p, items, ctas, box_rows, stream);
}
