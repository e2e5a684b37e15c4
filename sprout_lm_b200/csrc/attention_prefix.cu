// Attention of a step's tokens over the paged cache where requests hold the same leading pages, those pages' keys and values read once for
// all requests that hold them.
//
// A softmax over keys that are divided into ranges is put together from the ranges: with m_S the maximum of a range's scores, l_S the
// sum of e^(s - m_S) and o_S the sum of e^(s - m_S) v,   o = sum_S e^(m_S - m) o_S / sum_S e^(m_S - m) l_S,   m the largest m_S.
// So the keys that several requests share are a range of their own, whose rows are the tokens of all of them: a matrix product in place of
// as many passes over the same keys.  The requests' own keys are ranges of few rows, streams of keys and values.  Long ranges are
// divided again, so that the launch fills the device.
//
// The items' partial results come from attention_prefix_simple_kernel (CUDA cores, 32-bit products, any head size and either type), or, for
// bfloat16 and head sizes up to 128, from attention_prefix_mma_kernel (mma.sync), for few rows of most caches from
// attention_prefix_stream.cu and for many rows over whole pages from attention_prefix_tcgen05.cu; one launch adds them up.
#include <algorithm>
#include <atomic>

#include "attention_bf16.cuh"
#include "attention_prefix.cuh"

using namespace sprout_prefix;
using namespace sprout_attn;

namespace {

// ------------------------------------------------------------------ CUDA cores
// 16 rows, 64 keys at a time in shared memory as float32.  A thread has 2 rows x 4 keys of the scores, and 2 rows x 4 columns in
// every 64 of the output: six 16-byte reads of shared memory for 32 fused multiply-adds, which bound it.  21 tokens of 12 requests over 1,500
// shared keys and up to 200 own (14 heads over 2 of 64, float32): 14 us, the merge 7 behind it.
constexpr int SIMPLE_ROWS = 16, SIMPLE_KEYS = 64, SIMPLE_THREADS = 128;

__host__ __device__ constexpr int simple_width(int head_dim) { return (head_dim + 3) / 4 * 4; }
size_t simple_smem(int head_dim) {
  const size_t w = simple_width(head_dim);
  return ((w + 4) * (SIMPLE_KEYS + SIMPLE_ROWS) + w * SIMPLE_KEYS + SIMPLE_ROWS * (SIMPLE_KEYS + 4) + SIMPLE_ROWS * 3) * sizeof(float) + SIMPLE_KEYS * sizeof(long long);
}

// Four elements of a row from column c on, zero from head_dim on; FOURS: rows are whole fours and start on their boundaries.
template <bool FOURS> __device__ __forceinline__ float4 load_elements(const float* row, int c, int head_dim) {
  if (FOURS) return c < head_dim ? *(const float4*)(row + c) : make_float4(0.f, 0.f, 0.f, 0.f);
  return make_float4(c < head_dim ? row[c] : 0.f, c + 1 < head_dim ? row[c + 1] : 0.f, c + 2 < head_dim ? row[c + 2] : 0.f, c + 3 < head_dim ? row[c + 3] : 0.f);
}
template <bool FOURS> __device__ __forceinline__ float4 load_elements(const __nv_bfloat16* row, int c, int head_dim) {
  if (FOURS) {
    if (c >= head_dim) return make_float4(0.f, 0.f, 0.f, 0.f);
    const uint2 t = *(const uint2*)(row + c);
    return make_float4(__uint_as_float(t.x << 16), __uint_as_float(t.x & 0xffff0000u), __uint_as_float(t.y << 16), __uint_as_float(t.y & 0xffff0000u));
  }
  return make_float4(c < head_dim ? to_float(row[c]) : 0.f, c + 1 < head_dim ? to_float(row[c + 1]) : 0.f, c + 2 < head_dim ? to_float(row[c + 2]) : 0.f,
                     c + 3 < head_dim ? to_float(row[c + 3]) : 0.f);
}

// COLUMNS: of 64, that hold head_dim
template <typename T, int COLUMNS, bool FOURS>
__global__ void __launch_bounds__(SIMPLE_THREADS)
attention_prefix_simple_kernel(const Params p) {
  extern __shared__ __align__(16) float simple_shared[];
  const int w = simple_width(p.head_dim), ks = w + 4;
  long long* rows = (long long*)simple_shared;         // [64] element offsets, -1: no such key
  float* sK = (float*)(rows + SIMPLE_KEYS);            // [64][ks]
  float* sQ = sK + SIMPLE_KEYS * ks;                   // [16][ks]
  float* sV = sQ + SIMPLE_ROWS * ks;                   // [64][w]
  float* sP = sV + SIMPLE_KEYS * w;                    // [16][68]
  float* s_m = sP + SIMPLE_ROWS * (SIMPLE_KEYS + 4);   // [16] maxima, sums, what a pass multiplies the outputs by
  float* s_l = s_m + SIMPLE_ROWS;
  float* s_a = s_l + SIMPLE_ROWS;
  const Item planned = p.items[blockIdx.x];
  begin_items(p);
  const Item item = in_step(p, planned);
  const int g = blockIdx.y, group = p.heads / p.kv_heads, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int* table = p.block_table + (size_t)item.table * p.table_stride;
  // a thread keeps its four columns and walks down the rows
  constexpr int PIECES = 16 * COLUMNS, AT_ONCE = SIMPLE_THREADS / PIECES;
  const int own_c = tid % PIECES * 4, own_row = tid / PIECES;
#pragma unroll
  for (int i = own_row; i < SIMPLE_ROWS; i += AT_ONCE) {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (i < item.rows)
      v = load_elements<FOURS>((const T*)p.q + (size_t)p.order[place_of_row(item, i, group)] * p.q_stride + (size_t)head_of_row(item, i, group, g) * p.head_dim, own_c, p.head_dim);
    if (own_c < w) *(float4*)(sQ + i * ks + own_c) = v;
  }
  if (tid < SIMPLE_ROWS) { s_m[tid] = -INFINITY; s_l[tid] = 0.f; }
  const int r0 = tid / 16 * 2, c0 = tid % 16 * 4;
  float acc[2][COLUMNS][4];
#pragma unroll
  for (int a = 0; a < 2; a++)
#pragma unroll
    for (int b = 0; b < COLUMNS; b++)
#pragma unroll
      for (int c = 0; c < 4; c++) acc[a][b][c] = 0.f;
  for (int base = item.key_begin; base < item.key_end; base += SIMPLE_KEYS) {
    __syncthreads();                                   // the pass before is done with the keys and values
    if (tid < SIMPLE_KEYS) rows[tid] = base + tid < item.key_end ? key_row(p, table, base + tid, g) : -1;
    __syncthreads();
    if (own_c < w) {
      constexpr int BATCH = 8;                         // rows of keys and values on their way at a time
#pragma unroll
      for (int j0 = 0; j0 < SIMPLE_KEYS; j0 += BATCH * AT_ONCE) {
        float4 k[BATCH], v[BATCH];
#pragma unroll
        for (int j = 0; j < BATCH; j++) {
          const long long at = rows[j0 + j * AT_ONCE + own_row];
          k[j] = at >= 0 ? load_elements<FOURS>((const T*)p.k_cache + at, own_c, p.head_dim) : make_float4(0.f, 0.f, 0.f, 0.f);
          v[j] = at >= 0 ? load_elements<FOURS>((const T*)p.v_cache + at, own_c, p.head_dim) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int j = 0; j < BATCH; j++) {
          *(float4*)(sK + (j0 + j * AT_ONCE + own_row) * ks + own_c) = k[j];
          *(float4*)(sV + (j0 + j * AT_ONCE + own_row) * w + own_c) = v[j];
        }
      }
    }
    __syncthreads();
    float s[2][4] = {};
    for (int d = 0; d < w; d += 4) {
      float4 q[2], k[4];
#pragma unroll
      for (int a = 0; a < 2; a++) q[a] = *(const float4*)(sQ + (r0 + a) * ks + d);
#pragma unroll
      for (int b = 0; b < 4; b++) k[b] = *(const float4*)(sK + (tid % 16 + b * 16) * ks + d);
#pragma unroll
      for (int a = 0; a < 2; a++)
#pragma unroll
        for (int b = 0; b < 4; b++) s[a][b] = fmaf(q[a].x, k[b].x, fmaf(q[a].y, k[b].y, fmaf(q[a].z, k[b].z, fmaf(q[a].w, k[b].w, s[a][b]))));
    }
#pragma unroll
    for (int a = 0; a < 2; a++)
#pragma unroll
      for (int b = 0; b < 4; b++) sP[(r0 + a) * (SIMPLE_KEYS + 4) + tid % 16 + b * 16] = s[a][b] * p.scale_log2;
    __syncthreads();
    // softmax: a warp four rows, a lane two keys
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int r = warp * 4 + i;
      float* row = sP + r * (SIMPLE_KEYS + 4);
      const float x0 = rows[lane] >= 0 ? row[lane] : -INFINITY;
      const float x1 = rows[lane + 32] >= 0 ? row[lane + 32] : -INFINITY;
      const float before = s_m[r], m = fmaxf(before, warp_max(fmaxf(x0, x1)));
      const float e0 = x0 == -INFINITY ? 0.f : exp2f(x0 - m), e1 = x1 == -INFINITY ? 0.f : exp2f(x1 - m);
      const float sum = warp_sum(e0 + e1);
      row[lane] = e0;
      row[lane + 32] = e1;
      __syncwarp();
      if (lane == 0) {
        const float a = before == -INFINITY ? 0.f : exp2f(before - m);
        s_m[r] = m;
        s_l[r] = s_l[r] * a + sum;
        s_a[r] = a;
      }
      __syncwarp();
    }
    __syncthreads();
    const float a0 = s_a[r0], a1 = s_a[r0 + 1];
#pragma unroll
    for (int b = 0; b < COLUMNS; b++)
#pragma unroll
      for (int c = 0; c < 4; c++) { acc[0][b][c] *= a0; acc[1][b][c] *= a1; }
    for (int j = 0; j < SIMPLE_KEYS; j += 4) {
      float p0[4], p1[4];
      *(float4*)p0 = *(const float4*)(sP + r0 * (SIMPLE_KEYS + 4) + j);
      *(float4*)p1 = *(const float4*)(sP + (r0 + 1) * (SIMPLE_KEYS + 4) + j);
#pragma unroll
      for (int b = 0; b < COLUMNS; b++) {
        if (b * 64 + c0 >= w) break;
#pragma unroll
        for (int jj = 0; jj < 4; jj++) {
          const float4 v = *(const float4*)(sV + (j + jj) * w + b * 64 + c0);
          acc[0][b][0] = fmaf(p0[jj], v.x, acc[0][b][0]); acc[0][b][1] = fmaf(p0[jj], v.y, acc[0][b][1]);
          acc[0][b][2] = fmaf(p0[jj], v.z, acc[0][b][2]); acc[0][b][3] = fmaf(p0[jj], v.w, acc[0][b][3]);
          acc[1][b][0] = fmaf(p1[jj], v.x, acc[1][b][0]); acc[1][b][1] = fmaf(p1[jj], v.y, acc[1][b][1]);
          acc[1][b][2] = fmaf(p1[jj], v.z, acc[1][b][2]); acc[1][b][3] = fmaf(p1[jj], v.w, acc[1][b][3]);
        }
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int a = 0; a < 2; a++) {
    const int i = r0 + a;
    if (i >= item.rows) break;
    const size_t at = (size_t)(p.part_start[place_of_row(item, i, group)] + item.part) * p.heads + head_of_row(item, i, group, g);
#pragma unroll
    for (int b = 0; b < COLUMNS; b++)
#pragma unroll
      for (int c = 0; c < 4; c++) if (b * 64 + c0 + c < p.head_dim) p.part_out[at * p.head_dim + b * 64 + c0 + c] = acc[a][b][c];
    if (tid % 16 == 0) p.part_sum[at] = make_float2(s_m[i], s_l[i]);
  }
  end_items(p);
}

// ------------------------------------------------------------------ mma.sync
// Keys and values in steps through shared memory (cp.async), three or four CTAs an SM.  The next step's keys are asked for when this
// step's scores are done, its values when this step's outputs are, so that a buffer of each is always on its way or in use.  NARROW (an
// item of up to 16 rows): the rows are one tile of the MMA, each of the 4 warps takes 32 of a step's 128 keys, and the warps' results are
// merged at the end.  Else an item has up to 64 rows, 16 a warp, and every warp takes all 64 keys of a step.  What bounds a launch of few
// steps is their chain (fetch, scores, exponentials, products): 90 requests of a token or two over six prefixes of 2,500 to 5,000 keys (14
// heads over 2 of 64) take 15 us as 64-row items beside 9 for the requests' own keys.
constexpr int MMA_THREADS = 128;

template <int HD, bool NARROW>
struct MmaShape {
  static constexpr int ROWS = NARROW ? 16 : 64, KEYS = NARROW ? 128 : 64, STRIDE = HD + 8, CHUNK = NARROW ? 32 : 64;      // CHUNK: a warp's keys of a step
  static constexpr size_t SMEM = (size_t)(ROWS + 2 * KEYS) * STRIDE * 2 + 2 * KEYS * sizeof(long long);
  static constexpr int CTAS = HD > 96 ? 3 : 4;
};

template <int HD, bool NARROW>
__global__ void __launch_bounds__(MMA_THREADS, MmaShape<HD, NARROW>::CTAS)
attention_prefix_mma_kernel(const Params p) {
  using L = MmaShape<HD, NARROW>;
  constexpr int STRIDE = L::STRIDE, PIECES = HD / 8, CHUNK = L::CHUNK, KEYS = L::KEYS;
  extern __shared__ __align__(16) uint8_t mma_shared[];
  long long* rows = (long long*)mma_shared;            // [2][KEYS] element offsets of this step's keys and the next one's, -1: no such key
  __nv_bfloat16* sQ = (__nv_bfloat16*)(rows + 2 * KEYS);           // [ROWS][STRIDE]
  __nv_bfloat16* sK = sQ + L::ROWS * STRIDE;           // [KEYS][STRIDE]
  __nv_bfloat16* sV = sK + KEYS * STRIDE;
  const Item planned = p.items[blockIdx.x];
  begin_items(p);
  const Item item = in_step(p, planned);
  const int g = blockIdx.y, group = p.heads / p.kv_heads, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int* table = p.block_table + (size_t)item.table * p.table_stride;
  auto look_up = [&](int base) { return tid < KEYS && base + tid < item.key_end ? key_row(p, table, base + tid, g) : -1ll; };
  auto fetch = [&](__nv_bfloat16* to, const void* cache, const long long* at) {
#pragma unroll
    for (int k = 0; k < (KEYS * PIECES + MMA_THREADS - 1) / MMA_THREADS; k++) {
      const int idx = tid + k * MMA_THREADS, j = idx / PIECES, c = idx % PIECES;
      if (KEYS * PIECES % MMA_THREADS != 0 && j >= KEYS) break;
      const long long from = at[j];
      if (from >= 0) cp_async16(to + j * STRIDE + c * 8, (const __nv_bfloat16*)cache + from + c * 8);
      else *(uint4*)(to + j * STRIDE + c * 8) = make_uint4(0, 0, 0, 0);      // finite: its weight is zero, and zero times a NaN is not
    }
  };
  const long long mine = look_up(item.key_begin);
  // the query rows, their offsets first (in the room of the next step's): each is behind a read of its own
  if (tid < KEYS) rows[tid] = mine;
  if (tid < L::ROWS)
    rows[KEYS + tid] = tid < item.rows ? (long long)p.order[place_of_row(item, tid, group)] * p.q_stride + (long long)head_of_row(item, tid, group, g) * HD : -1;
  bool whole = __syncthreads_and(tid >= KEYS || mine >= 0);
  fetch(sK, p.k_cache, rows);
  cp_async_commit();
  fetch(sV, p.v_cache, rows);
  cp_async_commit();
  constexpr int EACH = (L::ROWS * PIECES + MMA_THREADS - 1) / MMA_THREADS;
  uint4 held[EACH];                                    // all on their way before the first is stored
#pragma unroll
  for (int k = 0; k < EACH; k++) {
    const int idx = tid + k * MMA_THREADS;
    const long long at = rows[KEYS + min(idx / PIECES, L::ROWS - 1)];
    held[k] = at >= 0 ? *(const uint4*)((const __nv_bfloat16*)p.q + at + idx % PIECES * 8) : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int k = 0; k < EACH; k++) {
    const int idx = tid + k * MMA_THREADS;
    if (idx < L::ROWS * PIECES) *(uint4*)(sQ + idx / PIECES * STRIDE + idx % PIECES * 8) = held[k];
  }
  const int tile = NARROW ? 0 : warp, gr = lane >> 2, qc = lane & 3, chunk = NARROW ? warp * CHUNK : 0;
  const int row0 = tile * 16 + gr, row1 = row0 + 8;    // of the item, this lane's in the fragments
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f, o[HD / 8][4];
#pragma unroll
  for (int n = 0; n < HD / 8; n++) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  int held_rows = 0;                                   // which half of `rows` this step's are in
  for (int base = item.key_begin; base < item.key_end; base += KEYS, held_rows ^= KEYS) {
    const bool more = base + KEYS < item.key_end, works = tile * 16 < item.rows && base + chunk < item.key_end;
    const long long next = more ? look_up(base + KEYS) : -1;
    cp_async_wait<1>();
    __syncthreads();                                   // the keys (and the query rows) are there
    float s[CHUNK / 8][4];
#pragma unroll
    for (int n = 0; n < CHUNK / 8; n++) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
    if (works) {
#pragma unroll
      for (int kk = 0; kk < HD / 16; kk++) {
        uint32_t a[4];
        ldmatrix_x4(a, sQ + (tile * 16 + (lane & 15)) * STRIDE + kk * 16 + (lane >> 4) * 8);
#pragma unroll
        for (int n = 0; n < CHUNK / 16; n++) {
          uint32_t b[4];                               // keys 16 n .. + 15: fragments of two MMAs
          ldmatrix_x4(b, sK + (chunk + n * 16 + (lane & 7) + ((lane >> 4) << 3)) * STRIDE + kk * 16 + ((lane >> 3) & 1) * 8);
          mma_bf16(s[2 * n], a, b[0], b[1]);
          mma_bf16(s[2 * n + 1], a, b[2], b[3]);
        }
      }
    }
    if (tid < KEYS) rows[(held_rows ^ KEYS) + tid] = next;
    const bool next_whole = __syncthreads_and(tid >= KEYS || next >= 0);      // all are done with the keys
    if (more) fetch(sK, p.k_cache, rows + (held_rows ^ KEYS));
    cp_async_commit();
    uint32_t pf[CHUNK / 16][4];                        // the weights as bfloat16, the A operand of P V
    float alpha0 = 1.f, alpha1 = 1.f;
    if (works) {
      float top0 = m0, top1 = m1;
#pragma unroll
      for (int n = 0; n < CHUNK / 8; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) s[n][i] *= p.scale_log2;
      if (!whole)
#pragma unroll
        for (int n = 0; n < CHUNK / 8; n++)
#pragma unroll
          for (int i = 0; i < 2; i++) if (rows[held_rows + chunk + n * 8 + qc * 2 + i] < 0) s[n][i] = s[n][2 + i] = -INFINITY;
#pragma unroll
      for (int n = 0; n < CHUNK / 8; n++) {
        top0 = fmaxf(top0, fmaxf(s[n][0], s[n][1]));
        top1 = fmaxf(top1, fmaxf(s[n][2], s[n][3]));
      }
      top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, 1));
      top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, 2));
      top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, 1));
      top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, 2));
      alpha0 = m0 == -INFINITY ? 0.f : exp2_fast(m0 - top0);
      alpha1 = m1 == -INFINITY ? 0.f : exp2_fast(m1 - top1);
      m0 = top0;
      m1 = top1;
      const float base0 = m0 == -INFINITY ? 0.f : m0, base1 = m1 == -INFINITY ? 0.f : m1;
      float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
      for (int n = 0; n < CHUNK / 8; n++) {
        const float e0 = exp2_fast(s[n][0] - base0), e1 = exp2_fast(s[n][1] - base0), e2 = exp2_fast(s[n][2] - base1), e3 = exp2_fast(s[n][3] - base1);
        sum0 += e0 + e1;
        sum1 += e2 + e3;
        pf[n >> 1][(n & 1) * 2] = pack_bf16(e0, e1);
        pf[n >> 1][(n & 1) * 2 + 1] = pack_bf16(e2, e3);
      }
      l0 = l0 * alpha0 + sum0;
      l1 = l1 * alpha1 + sum1;
#pragma unroll
      for (int n = 0; n < HD / 8; n++) { o[n][0] *= alpha0; o[n][1] *= alpha0; o[n][2] *= alpha1; o[n][3] *= alpha1; }
    }
    cp_async_wait<1>();
    __syncthreads();                                   // the values are there
    if (works) {
#pragma unroll
      for (int k = 0; k < CHUNK / 16; k++)
#pragma unroll
        for (int n = 0; n < HD / 16; n++) {
          uint32_t b[4];
          ldmatrix_x4_trans(b, sV + (chunk + k * 16 + (lane & 15)) * STRIDE + n * 16 + (lane >> 4) * 8);
          mma_bf16(o[2 * n], pf[k], b[0], b[1]);
          mma_bf16(o[2 * n + 1], pf[k], b[2], b[3]);
        }
    }
    __syncthreads();                                   // all are done with the values
    if (more) fetch(sV, p.v_cache, rows + (held_rows ^ KEYS));
    cp_async_commit();
    whole = next_whole;
  }
  cp_async_wait<0>();
  l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
  l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
  l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
  l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
  auto slot = [&](int i) { return (size_t)(p.part_start[place_of_row(item, i, group)] + item.part) * p.heads + head_of_row(item, i, group, g); };
  if (!NARROW) {
#pragma unroll
    for (int half = 0; half < 2; half++) {
      const int i = half ? row1 : row0;
      if (i >= item.rows) continue;
      const size_t at = slot(i);
#pragma unroll
      for (int n = 0; n < HD / 8; n++) *(float2*)(p.part_out + at * HD + n * 8 + qc * 2) = make_float2(o[n][half * 2], o[n][half * 2 + 1]);
      if (qc == 0) p.part_sum[at] = half ? make_float2(m1, l1) : make_float2(m0, l0);
    }
    end_items(p);
    return;
  }
  // the warps' results, in the keys' and values' room: [4 warps][16 rows][HD], maxima and sums behind them
  float* w_out = (float*)sK;
  float2* w_sum = (float2*)(w_out + 4 * 16 * HD);
  static_assert((size_t)4 * 16 * HD * 4 + 64 * 8 <= (size_t)2 * KEYS * STRIDE * 2 || !NARROW, "the warps' results fit the keys' and values' room");
  __syncthreads();
#pragma unroll
  for (int n = 0; n < HD / 8; n++) {
    *(float2*)(w_out + (warp * 16 + gr) * HD + n * 8 + qc * 2) = make_float2(o[n][0], o[n][1]);
    *(float2*)(w_out + (warp * 16 + gr + 8) * HD + n * 8 + qc * 2) = make_float2(o[n][2], o[n][3]);
  }
  if (qc == 0) { w_sum[warp * 16 + gr] = make_float2(m0, l0); w_sum[warp * 16 + gr + 8] = make_float2(m1, l1); }
  __syncthreads();
  for (int idx = tid; idx < item.rows * (HD / 4); idx += MMA_THREADS) {
    const int i = idx / (HD / 4), c = idx % (HD / 4) * 4;
    float2 ml[4];
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int w = 0; w < 4; w++) { ml[w] = w_sum[w * 16 + i]; m = fmaxf(m, ml[w].x); }
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < 4; w++) {
      const float f = ml[w].x == -INFINITY ? 0.f : exp2f(ml[w].x - m);
      const float4 t = *(const float4*)(w_out + (w * 16 + i) * HD + c);
      sum.x = fmaf(t.x, f, sum.x); sum.y = fmaf(t.y, f, sum.y); sum.z = fmaf(t.z, f, sum.z); sum.w = fmaf(t.w, f, sum.w);
      l = fmaf(ml[w].y, f, l);
    }
    const size_t at = slot(i);
    *(float4*)(p.part_out + at * HD + c) = sum;
    if (c == 0) p.part_sum[at] = make_float2(m, l);
  }
  end_items(p);
}

// ------------------------------------------------------------------ the parts of a row put together
// WARPS warps per (token, head), each of them every WARPS-th part, a lane two columns in every 64; the first warp also adds the keys of the
// member's own tokens that the items leave out, a lane a key.  One warp for a row of few parts; a row of 35 parts in one warp is a chain
// of five waits for memory.  What bounds it is those waits, and for many rows the parts' way out of L2: 128 tokens of 28 heads of 128 in 10
// parts 9.6 us behind the items.
// MERGE_FROM: parts a row, on average.  13 parts (64 tokens of 14 heads of 64): 16.7 us a call with four warps, 15.4 with one; 23 (29 tokens
// of 28 heads of 128): 20.3 and 23.2; 29 (11 tokens of 14 of 64): 9.0 and 10.3.
constexpr int MERGE_THREADS = 128, MERGE_SPLIT = 4, MERGE_FROM = 20;

template <typename T, int PAIRS, int WARPS>
__global__ void __launch_bounds__(MERGE_THREADS)
attention_prefix_merge_kernel(const Params p) {
  constexpr int ROWS = MERGE_THREADS / 32 / WARPS;     // of a block
  __shared__ float s_max[MERGE_THREADS / 32];
  __shared__ float s_sum[WARPS > 1 ? WARPS : 1][PAIRS * 64 + 1];
  pdl_launch_dependents();
  // What the items do not write is read before they are waited for: behind the gate, and the plan before it.
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, share = warp % WARPS, group = p.heads / p.kv_heads;
  const long long row = (long long)blockIdx.x * ROWS + warp / WARPS;
  if (row >= (long long)p.tokens * p.heads) return;    // whole blocks where warps share a row
  const int head = (int)(row % p.heads), place = (int)(row / p.heads), token = p.order[place], g = head / group;
  const int first = p.part_start[place], end = p.part_start[place + 1];
  // how far the step is behind the plan's own; outside what the plan serves it is another step's
  const int extra = share == 0 ? p.extra[place] : 0;
  int seen = p.seen[place];
  pass_gate(p);
  if (share == 0 && head == 0 && lane == 0) {
    const int ahead = p.positions[token] - (seen + extra - 1);
    if (ahead < 0 || ahead > p.stretch) atomicOr(p.status, SPROUT_STATUS_BAD_POSITION);        // a step that the plan does not serve
  }
  // where the member's further keys begin in this step
  if (p.stretch > 0 && extra > 0) seen += min(max(p.positions[token] - (seen + extra - 1), 0), p.stretch);
  float m = -INFINITY, l = 0.f, sum[PAIRS][2];
#pragma unroll
  for (int k = 0; k < PAIRS; k++) sum[k][0] = sum[k][1] = 0.f;
  float score = -INFINITY;                             // of this lane's extra key
  long long at = -1;
  if (extra > 0) {
    if (lane < extra) at = key_row(p, p.block_table + (size_t)p.table_of[place] * p.table_stride, seen + lane, g);
    const T* q = (const T*)p.q + (size_t)token * p.q_stride + (size_t)head * p.head_dim;
    for (int j = 0; j < extra; j++) {
      const long long k_at = __shfl_sync(0xffffffffu, at, j);
      if (k_at < 0) continue;
      float dot = 0.f;
#pragma unroll
      for (int k = 0; k < PAIRS; k++) {
        const int c = k * 64 + lane * 2;
        if (c < p.head_dim) dot = fmaf(to_float(q[c]), to_float(((const T*)p.k_cache)[k_at + c]), fmaf(to_float(q[c + 1]), to_float(((const T*)p.k_cache)[k_at + c + 1]), dot));
      }
      dot = warp_sum(dot);
      if (lane == j) score = dot * p.scale_log2;
    }
  }
  pdl_wait();
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.gate = 0;
  // the warp's parts, every WARPS-th: a lane the sums of one in every 32, and the outputs of the first AHEAD, all on their way at a time
  constexpr int AHEAD = PAIRS <= 2 ? 8 : 4;
  const int mine = (end - first - share + WARPS - 1) / WARPS;
  auto sums_of = [&](int i) { return i < mine ? __ldcg(&p.part_sum[(size_t)(first + share + i * WARPS) * p.heads + head]) : make_float2(-INFINITY, 0.f); };
  const float* from = p.part_out + ((size_t)(first + share) * p.heads + head) * p.head_dim;
  float2 t[AHEAD][PAIRS];
  auto fetch = [&](int part) {
#pragma unroll
    for (int i = 0; i < AHEAD; i++)
#pragma unroll
      for (int k = 0; k < PAIRS; k++) {
        const int c = k * 64 + lane * 2;
        t[i][k] = part + i < mine && c < p.head_dim ? __ldcg((const float2*)(from + (size_t)(part + i) * WARPS * p.heads * p.head_dim + c)) : make_float2(0.f, 0.f);
      }
  };
  float2 held = sums_of(lane);
  fetch(0);
  m = held.x;
  for (int i = 32 + lane; i < mine; i += 32) m = fmaxf(m, sums_of(i).x);
  m = warp_max(fmaxf(m, score));
  if (WARPS > 1) {                                     // the extra keys' may be the largest
    if (lane == 0) s_max[warp] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; w++) m = fmaxf(m, s_max[w]);
  }
  for (int base = 0; base < mine; base += 32) {        // 32 parts at a time, a lane a part's factor
    if (base > 0) held = sums_of(base + lane);
    const float factor = held.x == -INFINITY ? 0.f : exp2f(held.x - m);
    l = fmaf(held.y, factor, l);
    for (int part = base; part < min(base + 32, mine); part += AHEAD) {
      if (part > 0) fetch(part);
#pragma unroll
      for (int i = 0; i < AHEAD; i++) {
        const float f = __shfl_sync(0xffffffffu, factor, (part + i) & 31);
        if (part + i < mine)
#pragma unroll
          for (int k = 0; k < PAIRS; k++) { sum[k][0] = fmaf(t[i][k].x, f, sum[k][0]); sum[k][1] = fmaf(t[i][k].y, f, sum[k][1]); }
      }
    }
  }
  l = warp_sum(l);
  for (int j = 0; j < extra; j++) {
    const long long v_at = __shfl_sync(0xffffffffu, at, j);
    const float e = exp2f(__shfl_sync(0xffffffffu, score, j) - m);
    if (v_at < 0) continue;
#pragma unroll
    for (int k = 0; k < PAIRS; k++) {
      const int c = k * 64 + lane * 2;
      if (c < p.head_dim) {
        sum[k][0] = fmaf(e, to_float(((const T*)p.v_cache)[v_at + c]), sum[k][0]);
        sum[k][1] = fmaf(e, to_float(((const T*)p.v_cache)[v_at + c + 1]), sum[k][1]);
      }
    }
    l += e;
  }
  if (WARPS > 1) {
#pragma unroll
    for (int k = 0; k < PAIRS; k++) { s_sum[share][k * 64 + lane * 2] = sum[k][0]; s_sum[share][k * 64 + lane * 2 + 1] = sum[k][1]; }
    if (lane == 0) s_sum[share][PAIRS * 64] = l;
    __syncthreads();
    if (share != 0) return;
#pragma unroll
    for (int w = 1; w < WARPS; w++) {
#pragma unroll
      for (int k = 0; k < PAIRS; k++) { sum[k][0] += s_sum[w][k * 64 + lane * 2]; sum[k][1] += s_sum[w][k * 64 + lane * 2 + 1]; }
      l += s_sum[w][PAIRS * 64];
    }
  }
  const float inv = l != 0.f ? 1.0f / l : 0.f;         // no key at all (every page outside the pool): zero
  T* to = (T*)p.out + (size_t)token * p.out_stride + (size_t)head * p.head_dim;
#pragma unroll
  for (int k = 0; k < PAIRS; k++) {
    const int c = k * 64 + lane * 2;
    if (c < p.head_dim) { to[c] = from_float<T>(sum[k][0] * inv); to[c + 1] = from_float<T>(sum[k][1] * inv); }
  }
}

// ------------------------------------------------------------------ launches
template <typename T, int COLUMNS, bool FOURS>
int launch_simple(const Params& p, int items, cudaStream_t stream) {
  // CTAs that start while the call before still runs go where there is room, several to an SM that others have left: as much shared memory
  // each as lets an SM hold its share of them alone keeps them even.  21 tokens over 1,700 keys, calls one after the other: 17.2 us a call,
  // 22.7 without (16.6 and 16.4 in a capture); 4 requests of up to 3 over 4,000 and 1,000: 19.9 and 22.6; 16 of one token 24.8 and 24.3.
  constexpr size_t MOST = 200 * 1024;                  // of an SM's shared memory
  static_assert(((64 * COLUMNS + 4) * (SIMPLE_KEYS + SIMPLE_ROWS) + 64 * COLUMNS * SIMPLE_KEYS + SIMPLE_ROWS * (SIMPLE_KEYS + 4) + SIMPLE_ROWS * 3) * 4 + SIMPLE_KEYS * 8 <= MOST, "an item fits");
  if (reserve_shared<attention_prefix_simple_kernel<T, COLUMNS, FOURS>>(MOST, "attention_shared_prefix")) return 1;
  const long long each = ((long long)items * p.kv_heads + sprout_sm_count() - 1) / sprout_sm_count();
  const size_t bytes = std::max(simple_smem(p.head_dim), MOST / (size_t)each / 16 * 16);
  sprout_launch(attention_prefix_simple_kernel<T, COLUMNS, FOURS>, dim3(items, p.kv_heads), dim3(SIMPLE_THREADS), bytes, stream, p);
  return sprout_check_launch("attention_prefix_simple");
}
template <typename T, bool FOURS>
int launch_simple_any(const Params& p, int items, cudaStream_t stream) {
  if (p.head_dim <= 64) return launch_simple<T, 1, FOURS>(p, items, stream);
  if (p.head_dim <= 128) return launch_simple<T, 2, FOURS>(p, items, stream);
  return launch_simple<T, 4, FOURS>(p, items, stream);
}

template <int HD, bool NARROW>
int launch_mma(const Params& p, int items, cudaStream_t stream) {
  constexpr size_t bytes = MmaShape<HD, NARROW>::SMEM;
  if (reserve_shared<attention_prefix_mma_kernel<HD, NARROW>>(bytes, "attention_shared_prefix")) return 1;
  sprout_launch(attention_prefix_mma_kernel<HD, NARROW>, dim3(items, p.kv_heads), dim3(MMA_THREADS), bytes, stream, p);
  return sprout_check_launch("attention_prefix_mma");
}
template <bool NARROW>
int launch_mma_any(const Params& p, int items, cudaStream_t stream) {
  switch (p.head_dim) {
    case 16: return launch_mma<16, NARROW>(p, items, stream);
    case 32: return launch_mma<32, NARROW>(p, items, stream);
    case 48: return launch_mma<48, NARROW>(p, items, stream);
    case 64: return launch_mma<64, NARROW>(p, items, stream);
    case 80: return launch_mma<80, NARROW>(p, items, stream);
    case 96: return launch_mma<96, NARROW>(p, items, stream);
    case 112: return launch_mma<112, NARROW>(p, items, stream);
    case 128: return launch_mma<128, NARROW>(p, items, stream);
  }
  return sprout_fail("attention_shared_prefix: head_dim %d is not the tensor cores'", p.head_dim);
}

template <typename T, int WARPS>
int launch_merge(const Params& p, cudaStream_t stream) {
  constexpr int rows = MERGE_THREADS / 32 / WARPS;
  const long long blocks = ((long long)p.tokens * p.heads + rows - 1) / rows;
  SPROUT_REQUIRE(blocks <= 0x7fffffffLL, "attention_shared_prefix: too many tokens");
  if (p.head_dim <= 64) sprout_launch(attention_prefix_merge_kernel<T, 1, WARPS>, dim3((unsigned)blocks), dim3(MERGE_THREADS), 0, stream, p);
  else if (p.head_dim <= 128) sprout_launch(attention_prefix_merge_kernel<T, 2, WARPS>, dim3((unsigned)blocks), dim3(MERGE_THREADS), 0, stream, p);
  else sprout_launch(attention_prefix_merge_kernel<T, 4, WARPS>, dim3((unsigned)blocks), dim3(MERGE_THREADS), 0, stream, p);
  return sprout_check_launch("attention_prefix_merge");
}

}  // namespace

int sprout_attention_prefix_tc(const sprout_prefix::Params& p, int items, cudaStream_t stream);          // attention_prefix_tcgen05.cu
int sprout_attention_prefix_stream(const sprout_prefix::Params& p, int items, int ctas, cudaStream_t stream);      // attention_prefix_stream.cu
extern "C" int sprout_attention_prefix_tc_supported(int head_dim, int page_tokens);

// Whether bfloat16 items of this head size run on the tensor cores.
SPROUT_API int sprout_attention_prefix_mma_supported(int head_dim) { return head_dim % 16 == 0 && head_dim > 0 && head_dim <= 128; }

// What a plan is to its calls (kernels.py: _PrefixPlan): its arrays on the device; `simple_items` for the CUDA cores, or `matrix_items` of up
// to 256 rows, `narrow_items` of up to 16 (walked by `narrow_ctas` CTAs where they stream) and `wide_items` of up to 64; the partial results
// in all; and the sizes.
struct PrefixPlan {
  const Item* items;
  const int* order; const int* part_start; const int* seen; const int* extra; const int* table_of;
  int simple_items, matrix_items, narrow_items, narrow_ctas, wide_items, dtype, tokens, parts, heads, kv_heads, head_dim, page_tokens, stretch, unused;
};
static_assert(sizeof(PrefixPlan) == 6 * 8 + 14 * 4, "as ctypes lays it out");

// part_out holds parts * heads * head_dim floats, part_sum as many pairs as parts * heads; gate is a word of 64 bits, whatever is in it.
SPROUT_API int sprout_attention_prefix(const PrefixPlan* plan, const void* q, long long q_stride, const void* k_cache, const void* v_cache, const int* block_table, int table_stride,
                                       const int* positions, float* part_out, float* part_sum, unsigned long long* gate, void* out, long long out_stride, int num_pages, int* status, cudaStream_t stream) {
  SPROUT_REQUIRE(plan && q && k_cache && v_cache && block_table && positions && plan->items && plan->order && plan->part_start && plan->seen && plan->extra && plan->table_of && part_out &&
                 part_sum && gate && out && status, "attention_shared_prefix: null pointer");
  const int simple_items = plan->simple_items, matrix_items = plan->matrix_items, narrow_items = plan->narrow_items, narrow_ctas = plan->narrow_ctas, wide_items = plan->wide_items;
  const int dtype = plan->dtype, tokens = plan->tokens, parts = plan->parts, heads = plan->heads, kv_heads = plan->kv_heads, head_dim = plan->head_dim, page_tokens = plan->page_tokens;
  SPROUT_REQUIRE(tokens > 0 && parts > 0 && plan->stretch >= 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && kv_heads <= 65535 && head_dim > 0 && head_dim <= 256 && head_dim % 2 == 0 && page_tokens > 0 && num_pages > 0,
                 "attention_shared_prefix: bad sizes tokens=%d heads=%d/%d head_dim=%d page=%d", tokens, heads, kv_heads, head_dim, page_tokens);
  SPROUT_REQUIRE(simple_items >= 0 && matrix_items >= 0 && narrow_items >= 0 && wide_items >= 0 && (narrow_items == 0 || narrow_ctas > 0) && (simple_items > 0) != (matrix_items + narrow_items + wide_items > 0), "attention_shared_prefix: bad item counts");
  SPROUT_REQUIRE(dtype == SPROUT_F32 || dtype == SPROUT_BF16, "attention_shared_prefix: bad dtype %d", dtype);
  SPROUT_REQUIRE(((uintptr_t)part_out & 15) == 0 && ((uintptr_t)part_sum & 7) == 0 && ((uintptr_t)gate & 7) == 0, "attention_shared_prefix: the partial results must start on 16- and 8-byte boundaries");
  static std::atomic<uint32_t> calls{0};
  Params p{q, q_stride, k_cache, v_cache, block_table, table_stride, positions, plan->items, plan->order, plan->part_start, plan->seen, plan->extra, plan->table_of, part_out, (float2*)part_sum, out, out_stride,
           tokens, heads, kv_heads, head_dim, page_tokens, num_pages, 1.4426950408889634f / sqrtf((float)head_dim), status, plan->stretch, 1, gate, 0x7fd5acedull << 32 | calls.fetch_add(1, std::memory_order_relaxed)};
  if (simple_items > 0) {
    // rows that are whole fours on their boundaries
    const int row = dtype == SPROUT_F32 ? 16 : 8;
    const bool fours = head_dim % 4 == 0 && q_stride % 4 == 0 && (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache) & (row - 1)) == 0;
    if (dtype == SPROUT_F32 ? (fours ? launch_simple_any<float, true>(p, simple_items, stream) : launch_simple_any<float, false>(p, simple_items, stream))
                            : (fours ? launch_simple_any<__nv_bfloat16, true>(p, simple_items, stream) : launch_simple_any<__nv_bfloat16, false>(p, simple_items, stream))) return 1;
  } else {
    SPROUT_REQUIRE(dtype == SPROUT_BF16 && sprout_attention_prefix_mma_supported(head_dim), "attention_shared_prefix: these sizes run on the CUDA cores");
    SPROUT_REQUIRE(((uintptr_t)q & 15) == 0 && q_stride % 8 == 0 && ((uintptr_t)k_cache & 15) == 0 && ((uintptr_t)v_cache & 15) == 0,
                   "attention_shared_prefix: rows must start on 16-byte boundaries");
    if (matrix_items > 0) {
      if (sprout_attention_prefix_tc(p, matrix_items, stream)) return 1;
      p.first = 0;
    }
    p.items += matrix_items;
    if (wide_items > 0) {
      p.items += narrow_items;
      if (launch_mma_any<false>(p, wide_items, stream)) return 1;
      p.items -= narrow_items;
      p.first = 0;
    }
    if (narrow_items > 0) {
      const bool boxes = sprout_attention_prefix_tc_supported(head_dim, page_tokens) && (long long)num_pages * kv_heads * page_tokens <= 0x7fffffffLL;
      if (boxes ? sprout_attention_prefix_stream(p, narrow_items, narrow_ctas, stream) : launch_mma_any<true>(p, narrow_items, stream)) return 1;
    }
  }
  const bool split = parts >= (long long)MERGE_FROM * tokens;
  if (dtype == SPROUT_F32) return split ? launch_merge<float, MERGE_SPLIT>(p, stream) : launch_merge<float, 1>(p, stream);
  return split ? launch_merge<__nv_bfloat16, MERGE_SPLIT>(p, stream) : launch_merge<__nv_bfloat16, 1>(p, stream);
}
