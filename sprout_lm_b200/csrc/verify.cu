// Verification of drafted tokens against the target's probabilities, with given random numbers.
//
// Request r brings n drafted tokens x_0 .. x_{n-1} and n + 1 rows of target logits l_0 .. l_n (l_i is what the target says after the
// tokens before x_i), and, where a model drafted, n rows of its logits d_i.  With p = softmax(l / T) and q = softmax(d / T) (all of q on
// x_i where nothing drafted with probabilities):
//
//   x_i stands if all before it stand and u_i q_i(x_i) < p_i(x_i), u_i a given uniform number: with probability min(1, p_i / q_i);
//   at the first i that does not stand the token is drawn from max(p_i - q_i, 0), made to sum to 1; if all stand, from p_n.
//
// A draw is the inverse of the cumulative distribution at a given uniform number w_i: the lowest index whose running sum exceeds w_i
// times the total.  So the emitted tokens are distributed as the target's own.  T = 0: x_i stands if it is the lowest index of l_i's
// maximum; the token is the first row's argmax that was not drafted.
//
// A draw decides between neighbouring tokens by a sum over the vocabulary, and neighbours with probabilities of 1e-6 lie next to one
// another: a running sum that is off by 1e-7 would pick the neighbour once in some ten draws.  So the sums a draw is made from are 64-bit
// sums of 64-bit exponentials (`pow2`: 1e-12).  Those take 33 cycles of an SM's quarter a warp of logits (some 15 64-bit operations, two
// cycles each), 1.09 T a second, while memory delivers 1.6 T logits a second: only the row that is drawn from takes them.
//
// Whether a draft stands is decided by float32 exponentials.  A term 2^((v - max) c) has its difference, c = log2(e) / T and their product
// rounded, 2^-24 of the exponent each, then the hardware's 2^-22 and up to eight float32 additions: a row's sum is off by at most
// (3 d + 12) 2^-24 of itself, d the mean of (max - v) / T under the row's own probabilities.  d is 2 to 6 for wide rows, so that is 1 to 2e-6
// at the most; a model of the roundings gives 1e-8 to 1.3e-7 for 151,936 normal logits at T of 0.5 to 1.7.  A draft whose p and u q are
// closer than that may be decided either way.
//
// Three launches.  verify_rows_kernel: every row in pieces of PIECE logits, a warp each, their maxima and sums of exponentials (greedy:
// the maximum's first index).  verify_decide_kernel: a block per request merges its rows' pieces, a warp a row, and finds the first row
// that does not stand.  verify_sums_kernel: the 64-bit sums of that row's runs, a block each; where there are few, the request's last
// block to be done also finds the run in which the draw falls and looks through it, else a fourth launch does.
//
// The difference in one pass: max(p - q, 0) needs both rows' sums before a single element of it is known.  With a_j, b_j the
// exponentials and Za, Zb their sums, (p_j - q_j) Zb = a_j rho - b_j, rho = Zb / Za.  The float32 sums give rho to the above, and so the set
// of tokens where the difference is positive but for those within that of zero: the pass adds up a, b and, over that set, a and b again,
// from which the exact rho makes the difference's sums a run.  They are off by as much of p at the most, and tokens within the run
// that the draw falls in are told apart exactly.  Where p and q are so close that this is much of the difference, a draft falls as seldom:
// what is emitted is off by no more than that.
#include "common.cuh"

namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int PER_THREAD = 16, RUN = THREADS * PER_THREAD;       // logits of a run
// The first kernel: blocks an SM, pieces that a warp takes at most, logits of a piece.  616 rows of 152,064 (a third of the drafts' greedy and
// not read, 320 MB): 71 us; 3 blocks an SM 76, 16 pieces a warp 79, pieces of 512 logits in 4 blocks 71 but 10 % more in what merges them.
constexpr int ROW_BLOCKS = 2, MAX_ITEMS = 8, PIECE = 1024;
constexpr int DRAW_THREADS = 512;          // of a block that draws and did not sum
constexpr int MAX_HELD = 256;              // runs whose sums the drawing block keeps in shared memory

struct PieceSum { double sum; float max; int index; int bad; int pad; };     // sum: of 2^((v - max) log2(e) / T)

// 2^y for y <= 0 to 1e-12: y = k + f with |f| <= 1/2, 2^f by a polynomial through the Chebyshev nodes, k into the exponent.
// Below 2^-1000 it is zero.
__device__ __forceinline__ double pow2(double y) {
  const double magic = 6755399441055744.0;             // 1.5 * 2^52: the sum's low bits are y rounded to a whole number
  const double t = y + magic;
  const double f = y - (t - magic);
  double p = 1.325497460306718e-06;
  p = fma(p, f, 1.5310078272506085e-05);
  p = fma(p, f, 0.00015403457039410448);
  p = fma(p, f, 0.0013333450572386462);
  p = fma(p, f, 0.009618129157656703);
  p = fma(p, f, 0.055504109412013614);
  p = fma(p, f, 0.24022650695821093);
  p = fma(p, f, 0.6931471805459344);
  p = fma(p, f, 1.0);
  const int k = __double2loint(t);
  const double r = __hiloint2double(__double2hiint(p) + (k << 20), __double2loint(p));
  return y >= -1000.0 ? r : 0.0;
}

__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ void better(float& v, int& i, float ov, int oi) {
  if (ov > v || (ov == v && oi < i)) { v = ov; i = oi; }
}

// The run's place of a thread's logit i: side by side in fours over the threads, so that a warp reads whole lines.
__device__ __forceinline__ int place_of(int i) { return (i >> 2) * (THREADS * 4) + (int)threadIdx.x * 4 + (i & 3); }
// Four logits from `at` on, -inf from `end` on.
__device__ __forceinline__ float4 load_four(const float* row, int at, int end, bool aligned) {
  if (aligned && at + 4 <= end) return *(const float4*)(row + at);
  return make_float4(at < end ? row[at] : -INFINITY, at + 1 < end ? row[at + 1] : -INFINITY, at + 2 < end ? row[at + 2] : -INFINITY,
                     at + 3 < end ? row[at + 3] : -INFINITY);
}
// A run's logits of this thread.
__device__ __forceinline__ void load_run(const float* run, int count, float (&v)[PER_THREAD]) {
  const bool aligned = ((uintptr_t)run & 15) == 0;
#pragma unroll
  for (int i = 0; i < PER_THREAD; i += 4) {
    const float4 t = load_four(run, place_of(i), count, aligned);
    v[i] = t.x; v[i + 1] = t.y; v[i + 2] = t.z; v[i + 3] = t.w;
  }
}

// What verify_decide_kernel leaves for a request's draw.
struct Chosen {
  int row;                                             // of the logits, -1: nothing is drawn
  int draft_row;                                       // whose probabilities are taken away, -1: none
  int without;                                         // a token that is left out, -1: none
  float top, top_q;                                    // the rows' maxima
  unsigned done;                                       // blocks of the draw whose sums are there
  double c, rho;                                       // log2(e) / T; the ratio of the rows' sums, from the float32 ones
};

// 64-bit sums of a run of the row that is drawn from: the exponentials of the target's and the draft's logits, and both again over the
// tokens where the difference is positive.
struct __align__(16) Sums { double a, b, above_a, above_b; };

struct Args {
  const float* logits; const float* draft_logits;      // [rows, vocab], [draft_rows, vocab]
  long long ld, draft_ld;
  const int* row_start; const float* temperature;      // [requests + 1], [requests] (null: 0)
  const int* drafts; const float* accept; const float* draw;      // [rows]
  int* out; int* accepted; int* status;                // [rows], [requests]
  PieceSum* pieces;                                    // [rows + draft_rows, per_row]
  Chosen* chosen; Sums* sums;                          // [requests], [requests, runs]
  int rows, draft_rows, requests, vocab, per_row, runs;            // pieces and runs of a row
  int items;                                           // pieces that a warp of the first kernel takes
  int fill;                                            // out holds nothing yet: -1 where no request writes
};

// The temperature of the request that row `row` (a draft row from p.rows on) belongs to: the last whose rows (draft rows: one fewer
// per request before) begin at or before it.  A warp asks 32 places at once.
__device__ __forceinline__ float temperature_of(const Args& p, int row) {
  if (p.temperature == nullptr) return 0.f;
  const int lane = threadIdx.x & 31, draft = row >= p.rows, own = draft ? row - p.rows : row;
  int lo = 0;
  for (int n = p.requests; n > 1;) {
    const int step = (n + 31) / 32, i = lo + lane * step;
    const bool before = lane * step < n && p.row_start[i] - (draft ? i : 0) <= own;
    const int last = max(0, 31 - __clz(__ballot_sync(0xffffffffu, before)));
    n = min(step, n - last * step);
    lo += last * step;
  }
  return p.temperature[lo];
}

// A warp takes `items` pieces one after the other, the next on its way while one is added up: no warp waits for another (a block a
// piece of 4,096 with barriers in its sums kept 3.7 TB/s in flight).  What bounds it is memory; an element takes some five
// instructions: its share of a load, of a maximum and a minimum of three, a difference, a product, the exponential and the sum.
__global__ void __launch_bounds__(THREADS, ROW_BLOCKS)
verify_rows_kernel(const Args p) {
  constexpr int LOGITS = PIECE / 32;                   // a lane's, in fours side by side over the lanes
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (p.fill) for (long long i = (long long)blockIdx.x * THREADS + threadIdx.x; i < p.rows; i += (long long)gridDim.x * THREADS) p.out[i] = -1;
  const long long all = (long long)(p.rows + p.draft_rows) * p.per_row, first = ((long long)blockIdx.x * WARPS + warp) * p.items;
  if (first >= all) return;
  const int items = (int)min((long long)p.items, all - first);
  int row = (int)(first / p.per_row), piece = (int)(first % p.per_row);
  auto place = [&](int i) { return (i >> 2) * 128 + lane * 4 + (i & 3); };
  // the piece is wanted: not of a greedy request's draft, whose probabilities nobody asks for
  auto fetch = [&](float temp, float (&v)[LOGITS]) {
    const bool draft = row >= p.rows;
    if (draft && !(temp > 0.f)) return;
    const float* base = (draft ? p.draft_logits + (size_t)(row - p.rows) * p.draft_ld : p.logits + (size_t)row * p.ld) + piece * PIECE;
    const int count = min(PIECE, p.vocab - piece * PIECE);
    const bool aligned = ((uintptr_t)base & 15) == 0;
#pragma unroll
    for (int i = 0; i < LOGITS; i += 4) {
      const float4 t = load_four(base, place(i), count, aligned);
      v[i] = t.x; v[i + 1] = t.y; v[i + 2] = t.z; v[i + 3] = t.w;
    }
  };
  float temp = 1.f, even[LOGITS], odd[LOGITS];
  fetch(temp, even);                                   // before it is known whether it is wanted: the question takes as long as the answer
  temp = temperature_of(p, row);
  auto step = [&](const float (&v)[LOGITS], float (&next)[LOGITS], bool more) {
    const int at_row = row, begin = piece * PIECE, count = min(PIECE, p.vocab - begin);
    const size_t slot = (size_t)row * p.per_row + piece;
    const float own_temp = temp;
    if (++piece == p.per_row) {
      piece = 0;
      row++;
      if (more) temp = temperature_of(p, row);
    }
    if (more) fetch(temp, next);
    const bool greedy = !(own_temp > 0.f);
    if (greedy && at_row >= p.rows) return;
    float best = -INFINITY, low = INFINITY;            // NaN is met below
    if (count == PIECE) {
#pragma unroll
      for (int i = 0; i < LOGITS; i += 2) {
        asm("max.f32 %0, %0, %1, %2;" : "+f"(best) : "f"(v[i]), "f"(v[i + 1]));
        asm("min.f32 %0, %0, %1, %2;" : "+f"(low) : "f"(v[i]), "f"(v[i + 1]));
      }
    } else {
#pragma unroll
      for (int i = 0; i < LOGITS; i++) {
        best = fmaxf(best, v[i]);                      // beyond the vocabulary: -inf
        if (place(i) < count) low = fminf(low, v[i]);
      }
    }
    best = warp_max(best);
    bool bad = __any_sync(0xffffffffu, !(low > -INFINITY)) || !(best < INFINITY);
    int index = 0x7fffffff;
    double sum = 0.0;
    if (greedy) {
#pragma unroll
      for (int i = LOGITS - 1; i >= 0; i--) {          // places rise with i
        bad |= v[i] != v[i];
        if (v[i] == best) index = begin + place(i);
      }
      index = __reduce_min_sync(0xffffffffu, index);
    } else {
      // infinite, it would make NaN of the maximum
      const float c = fminf((float)(1.4426950408889634 / (double)own_temp), 3e38f);
      float sums[4] = {0.f, 0.f, 0.f, 0.f};
      if (count == PIECE) {
#pragma unroll
        for (int i = 0; i < LOGITS; i++) sums[i & 3] += exp2_fast((v[i] - best) * c);
      } else {
#pragma unroll
        for (int i = 0; i < LOGITS; i++) if (place(i) < count) sums[i & 3] += exp2_fast((v[i] - best) * c);
      }
      sum = warp_sum_d((double)(sums[0] + sums[1]) + (double)(sums[2] + sums[3]));
      bad |= sum != sum;                               // a NaN among the logits
    }
    bad = __any_sync(0xffffffffu, bad);
    if (lane == 0) p.pieces[slot] = PieceSum{sum, best, index, bad, 0};
  };
  for (int item = 0; item < items; item += 2) {
    step(even, odd, item + 1 < items);
    if (item + 1 < items) step(odd, even, item + 2 < items);
  }
}

// What a row's pieces add up to: its maximum, first index and (with `sums`) sum relative to the maximum, in every lane of the warp.
struct RowSum { double sum; float max; int index; int bad; };
__device__ __forceinline__ RowSum merge_pieces(const PieceSum* pieces, int count, bool sums, double c) {
  constexpr int HELD = 8;                              // of a lane, all on their way at a time
  const int lane = threadIdx.x & 31;
  RowSum row{0.0, -INFINITY, 0x7fffffff, 0};
  for (int base = 0; base < count; base += 32 * HELD) {
    PieceSum held[HELD];
#pragma unroll
    for (int k = 0; k < HELD; k++) {
      const int i = base + k * 32 + lane;
      held[k] = i < count ? pieces[i] : PieceSum{0.0, -INFINITY, 0x7fffffff, 0, 0};
    }
    float best = row.max;
    int index = row.index, bad = row.bad;
#pragma unroll
    for (int k = 0; k < HELD; k++) {
      better(best, index, held[k].max, held[k].index);
      bad |= held[k].bad;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) better(best, index, __shfl_xor_sync(0xffffffffu, best, o), __shfl_xor_sync(0xffffffffu, index, o));
    double sum = 0.0;
    if (sums) {
#pragma unroll
      for (int k = 0; k < HELD; k++) if (held[k].sum > 0.0) sum += held[k].sum * pow2(((double)held[k].max - (double)best) * c);
      sum = warp_sum_d(sum);
      if (row.sum > 0.0) sum += row.sum * pow2(((double)row.max - (double)best) * c);
    }
    row = RowSum{sum, best, index, __any_sync(0xffffffffu, bad)};
  }
  return row;
}

__global__ void __launch_bounds__(THREADS)
verify_decide_kernel(const Args p) {
  __shared__ double s_z[WARPS], s_zq[WARPS];
  __shared__ float s_m[WARPS], s_mq[WARPS];
  __shared__ int s_best[WARPS], s_code[WARPS];         // per row of a batch: 0 stands, 1 does not, 2 and more: flagged
  pdl_launch_dependents();
  pdl_wait();
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int first = p.row_start[r], end = p.row_start[r + 1], count = end - first;
  if (first < 0 || end > p.rows || end <= first || (p.draft_rows > 0 && (first - r < 0 || end - r - 1 > p.draft_rows))) {
    if (tid == 0) { atomicOr(p.status, SPROUT_STATUS_BAD_ROWS); p.accepted[r] = -1; p.chosen[r].row = -1; }
    return;
  }
  const float temp = p.temperature ? p.temperature[r] : 0.f;
  const bool greedy = !(temp > 0.f);
  const double c = greedy ? 0.0 : 1.4426950408889634 / (double)temp;
  int row = 0, code = 0;
  for (int base = 0; base < count; base += WARPS) {
    const int i = base + warp;
    if (i < count) {
      const int x = i < count - 1 ? p.drafts[first + i] : 0, d = first - r + i;
      const bool token = x >= 0 && x < p.vocab, model = p.draft_rows > 0 && i < count - 1;
      const float u = greedy ? 0.f : p.accept[first + i];
      // asked for before the runs are merged: a read that waits for another
      const float lx = token ? p.logits[(size_t)(first + i) * p.ld + x] : 0.f, dx = token && model && !greedy ? p.draft_logits[(size_t)d * p.draft_ld + x] : 0.f;
      const RowSum s = merge_pieces(p.pieces + (size_t)(first + i) * p.per_row, p.per_row, !greedy, c);
      int verdict = s.bad ? SPROUT_STATUS_NONFINITE : 1;           // the last row never "stands": the draw is made there
      double zq = 0.0;
      float mq = 0.f;
      if (i < count - 1 && !s.bad) {
        if (!token) {
          verdict = SPROUT_STATUS_BAD_TOKEN;
        } else if (greedy) {
          verdict = x == s.index ? 0 : 1;
        } else {
          const double px = pow2(((double)lx - (double)s.max) * c) / s.sum;
          double qx = 1.0;
          if (model) {
            const RowSum t = merge_pieces(p.pieces + (size_t)(p.rows + d) * p.per_row, p.per_row, true, c);
            if (t.bad) verdict = SPROUT_STATUS_NONFINITE;
            zq = t.sum; mq = t.max;
            qx = pow2(((double)dx - (double)mq) * c) / zq;
          }
          if (verdict == 1) verdict = (double)u * qx < px ? 0 : 1;
        }
      }
      if (lane == 0) { s_z[warp] = s.sum; s_m[warp] = s.max; s_best[warp] = s.index; s_zq[warp] = zq; s_mq[warp] = mq; s_code[warp] = verdict; }
    }
    __syncthreads();
    int w = 0;
    while (w < WARPS && base + w < count && s_code[w] == 0) w++;
    row = base + w;
    if (w < WARPS && row < count) { code = s_code[w]; break; }
    __syncthreads();
  }
  const int slot = row % WARPS;                        // batches start at multiples of WARPS
  const bool draws = code <= 1 && !greedy, fell = row < count - 1;
  for (int i = tid; i < count; i += THREADS)
    if (i != row || !draws) p.out[first + i] = i < row ? p.drafts[first + i] : i == row && code <= 1 ? s_best[slot] : -1;
  if (tid == 0) {
    p.accepted[r] = row;
    if (code > 1) atomicOr(p.status, code);
    const bool difference = fell && p.draft_rows > 0;
    p.chosen[r] = Chosen{draws ? first + row : -1, difference ? first - r + row : -1, fell && !difference ? p.drafts[first + row] : -1,
                         s_m[slot], s_mq[slot], 0, c, difference ? s_zq[slot] / s_z[slot] : 0.0};
  }
}

// The run's sums of this block, by a thread per sum, the first four.
template <bool COUNTED>
__device__ __forceinline__ void sum_run(const Args& p, const Chosen& at, int run, Sums* to) {
  __shared__ Sums s_sums[WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int begin = run * RUN, count = min(RUN, p.vocab - begin);
  const bool difference = at.draft_row >= 0;
  float v[PER_THREAD], d[PER_THREAD];
  load_run(p.logits + (size_t)at.row * p.ld + begin, count, v);
  if (difference) load_run(p.draft_logits + (size_t)at.draft_row * p.draft_ld + begin, count, d);
  const double top = (double)at.top, top_q = (double)at.top_q;
  Sums sum = {0.0, 0.0, 0.0, 0.0};
  if (difference) {
#pragma unroll
    for (int i = 0; i < PER_THREAD; i++) {
      const double ea = pow2(((double)v[i] - top) * at.c), eb = pow2(((double)d[i] - top_q) * at.c);
      if (count == RUN || place_of(i) < count) {
        sum.a += ea;
        sum.b += eb;
        if (ea * at.rho > eb) { sum.above_a += ea; sum.above_b += eb; }
      }
    }
    sum.b = warp_sum_d(sum.b);
    sum.above_a = warp_sum_d(sum.above_a);
    sum.above_b = warp_sum_d(sum.above_b);
  } else {
#pragma unroll
    for (int i = 0; i < PER_THREAD; i++) {
      const double ea = pow2(((double)v[i] - top) * at.c);
      if ((count == RUN || place_of(i) < count) && begin + place_of(i) != at.without) sum.a += ea;
    }
  }
  sum.a = warp_sum_d(sum.a);
  if (lane == 0) s_sums[warp] = sum;
  __syncthreads();
  if (tid < 4) {
    double total = 0.0;
#pragma unroll
    for (int w = 0; w < WARPS; w++) total += ((const double*)&s_sums[w])[tid];
    ((double*)to)[tid] = total;
    if (COUNTED) {                                     // there before the block counts as done
      __threadfence();
      __syncwarp(0xf);
    }
  }
}

// A request's draw, by a block of N threads: from the sums of its runs, the run in which it falls, then its place there.
template <int N>
__device__ __forceinline__ void draw_token(const Args& p, const Chosen& at, const Sums* sums, int* out) {
  constexpr int LOGITS = RUN / N;
  __shared__ double s_sum[N / 32], s_before, s_target, s_rho;
  __shared__ int s_run, s_from_p, s_first, s_last;
  __shared__ Sums s_sums[MAX_HELD];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (p.runs <= MAX_HELD) {                            // gone through three times
    for (int i = tid; i < p.runs * 2; i += N) ((double2*)s_sums)[i] = __ldcg((const double2*)sums + i);
    __syncthreads();
    sums = s_sums;
  }
  if (warp == 0) {
    // the run in which the draw falls, a lane a run
    double rho = 1.0, total = 0.0;
    bool from_p = at.draft_row < 0;
    if (!from_p) {
      double za = 0.0, zb = 0.0;
      for (int i = lane; i < p.runs; i += 32) { za += sums[i].a; zb += sums[i].b; }
      rho = warp_sum_d(zb) / warp_sum_d(za);
    }
    auto weight = [&](int i) { return i >= p.runs ? 0.0 : from_p ? sums[i].a : fmax(0.0, fma(sums[i].above_a, rho, -sums[i].above_b)); };
    for (int attempt = 0; attempt < 2; attempt++) {
      total = 0.0;
      for (int i = lane; i < p.runs; i += 32) total += weight(i);
      total = warp_sum_d(total);
      if (from_p || total > 0.0) break;
      from_p = true;                                   // p and q are the same everywhere (what falls then fell by rounding): drawn from p
    }
    const double target = (double)p.draw[at.row] * total;
    double passed = 0.0, before = 0.0;
    int run = -1;                                      // stays so where the token that is left out has all the weight there is
    bool falls = false;
    for (int base = 0; base < p.runs && !falls; base += 32) {
      const double w = weight(base + lane);
      double upto = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double other = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += other;
      }
      const unsigned any = __ballot_sync(0xffffffffu, w > 0.0), over = __ballot_sync(0xffffffffu, w > 0.0 && passed + upto > target);
      if (any) {                                       // the first run that passes the target, or (so far) the last with any weight
        falls = over != 0;
        const int l = falls ? __ffs(over) - 1 : 31 - __clz(any);
        run = base + l;
        before = __shfl_sync(0xffffffffu, passed + upto - w, l);
      }
      passed += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane == 0) { s_run = run; s_before = before; s_target = target; s_rho = rho; s_from_p = from_p; s_first = 0x7fffffff; s_last = -1; }
  }
  __syncthreads();
  const int run = s_run;
  if (run < 0) {
    if (tid == 0) *out = at.without;
    return;
  }
  const bool from_p = s_from_p != 0;
  const double top = (double)at.top, top_q = (double)at.top_q, rho = s_rho, target = s_target;
  const int begin = run * RUN, count = min(RUN, p.vocab - begin);
  const float* logits = p.logits + (size_t)at.row * p.ld + begin;
  const float* draft = from_p ? nullptr : p.draft_logits + (size_t)at.draft_row * p.draft_ld + begin;
  const bool aligned = ((uintptr_t)logits & 15) == 0, aligned_q = ((uintptr_t)draft & 15) == 0;
  float v[LOGITS], d[LOGITS];
#pragma unroll
  for (int i = 0; i < LOGITS; i += 4) {           // side by side in every thread
    const int place = tid * LOGITS + i;
    const float4 t = load_four(logits, place, count, aligned), q = from_p ? t : load_four(draft, place, count, aligned_q);
    v[i] = t.x; v[i + 1] = t.y; v[i + 2] = t.z; v[i + 3] = t.w;
    d[i] = q.x; d[i + 1] = q.y; d[i + 2] = q.z; d[i + 3] = q.w;
  }
  double w[LOGITS], own = 0.0;
#pragma unroll
  for (int i = 0; i < LOGITS; i++) {
    const int place = tid * LOGITS + i;
    double e = pow2(((double)v[i] - top) * at.c);
    if (!from_p) e = fmax(0.0, fma(e, rho, -pow2(((double)d[i] - top_q) * at.c)));
    w[i] = place < count && begin + place != at.without ? e : 0.0;
    own += w[i];
  }
  double sum = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double other = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += other;
  }
  if (lane == 31) s_sum[warp] = sum;
  __syncthreads();
  double running = s_before;
  for (int i = 0; i < warp; i++) running += s_sum[i];
  running += sum - own;
  int first = 0x7fffffff, last = -1;
#pragma unroll
  for (int i = 0; i < LOGITS; i++) {
    running += w[i];
    if (w[i] > 0.0) {
      last = begin + tid * LOGITS + i;
      if (running > target && first == 0x7fffffff) first = last;
    }
  }
  if (first != 0x7fffffff) atomicMin(&s_first, first);
  if (last >= 0) atomicMax(&s_last, last);
  __syncthreads();
  if (tid == 0) *out = s_first != 0x7fffffff ? s_first : s_last;      // none by rounding: the last with any weight
}

// FEW: the request's last block to be done draws.
template <bool FEW>
__global__ void __launch_bounds__(THREADS, FEW ? 2 : 3)
verify_sums_kernel(const Args p) {
  __shared__ int s_draws;
  pdl_launch_dependents();
  pdl_wait();
  const int r = blockIdx.x / p.runs;
  const Chosen at = p.chosen[r];
  if (at.row < 0) return;
  sum_run<FEW>(p, at, blockIdx.x % p.runs, p.sums + blockIdx.x);
  if (!FEW) return;
  if (threadIdx.x == 0) s_draws = atomicAdd(&p.chosen[r].done, 1u) == (unsigned)p.runs - 1;
  __syncthreads();
  if (!s_draws) return;
  __threadfence();                                     // the other blocks' sums
  draw_token<THREADS>(p, at, p.sums + (size_t)r * p.runs, p.out + at.row);
}

__global__ void __launch_bounds__(DRAW_THREADS)
verify_draw_kernel(const Args p) {
  pdl_launch_dependents();
  pdl_wait();
  const Chosen at = p.chosen[blockIdx.x];
  if (at.row >= 0) draw_token<DRAW_THREADS>(p, at, p.sums + (size_t)blockIdx.x * p.runs, p.out + at.row);
}

}  // namespace

namespace {
int pieces_of(int vocab) { return (vocab + PIECE - 1) / PIECE; }
int runs_of(int vocab) { return (vocab + RUN - 1) / RUN; }
long long aligned16(long long bytes) { return (bytes + 15) & ~15LL; }
}  // namespace

static_assert(sizeof(Sums) == 32 && alignof(Sums) == 16 && sizeof(Chosen) % 8 == 0 && sizeof(PieceSum) % 8 == 0, "the scratch's parts start on their boundaries");

// Bytes of scratch, 16-byte aligned, for `rows` rows (target's and draft's together) of `vocab` logits.
SPROUT_API long long sprout_verify_scratch_bytes(int rows, int requests, int vocab) {
  return aligned16(rows * (long long)pieces_of(vocab) * (long long)sizeof(PieceSum)) + aligned16(requests * (long long)sizeof(Chosen)) +
         requests * (long long)runs_of(vocab) * (long long)sizeof(Sums);
}

// Request r's rows are row_start[r] .. row_start[r + 1] - 1 of `logits` [rows, vocab], at least one; its draft rows, one fewer, begin at
// row_start[r] - r of `draft_logits` (null with draft_rows 0: the drafts have no distribution).  Rows of `out` that are no request's, or of one
// that is flagged for its rows, become -1 with `fill` and stay as they are without.  temperature, accept and draw may be null
// together (all requests greedy).  Row i of `drafts` is the token drafted after row i's place; a request's last is not read.
SPROUT_API int sprout_verify(const float* logits, long long ld, const float* draft_logits, long long draft_ld, const int* drafts, const int* row_start,
                             const float* temperature, const float* accept, const float* draw, int* out, int fill, int* accepted, void* scratch,
                             int rows, int draft_rows, int requests, int vocab, int* status, cudaStream_t stream) {
  SPROUT_REQUIRE(rows > 0 && requests > 0 && requests <= rows && vocab > 0 && vocab <= 1 << 30 && ld >= 0, "verify: bad sizes rows=%d requests=%d vocab=%d ld=%lld", rows, requests, vocab, ld);
  SPROUT_REQUIRE(draft_rows == 0 || (draft_rows == rows - requests && draft_logits && draft_ld >= 0), "verify: a draft row per drafted token");
  SPROUT_REQUIRE(logits && drafts && row_start && out && accepted && scratch && status, "verify: null pointer");
  SPROUT_REQUIRE(((uintptr_t)scratch & 15) == 0, "verify: scratch must start on a 16-byte boundary");
  SPROUT_REQUIRE((temperature == nullptr) == (accept == nullptr) && (accept == nullptr) == (draw == nullptr), "verify: temperatures and both kinds of uniform numbers go together");
  const long long per_row = pieces_of(vocab), runs = runs_of(vocab), all = per_row * (rows + (long long)draft_rows);
  SPROUT_REQUIRE(rows + (long long)draft_rows <= 0x7fffffffLL && runs * requests <= 0x7fffffffLL, "verify: too many rows");
  Args p{logits, draft_logits, ld, draft_ld, row_start, temperature, drafts, accept, draw, out, accepted, status, nullptr, nullptr, nullptr,
         rows, draft_rows, requests, vocab, (int)per_row, (int)runs, 0, fill};
  uint8_t* at = (uint8_t*)scratch;
  p.pieces = (PieceSum*)at;
  at += aligned16(all * (long long)sizeof(PieceSum));
  p.chosen = (Chosen*)at;
  at += aligned16(requests * (long long)sizeof(Chosen));
  p.sums = (Sums*)at;
  // few pieces: a warp each; many: MAX_ITEMS of them, so that warps whose rows nobody asks for leave their place to others
  const long long warps = (long long)ROW_BLOCKS * WARPS * sprout_sm_count(), even = (all + warps - 1) / warps, items = even < MAX_ITEMS ? even : MAX_ITEMS;
  const long long blocks = (all + items * WARPS - 1) / (items * WARPS);
  SPROUT_REQUIRE(blocks <= 0x7fffffffLL, "verify: too many rows");
  p.items = (int)items;
  sprout_launch(verify_rows_kernel, dim3((unsigned)blocks), dim3(THREADS), 0, stream, p);
  if (sprout_check_launch("verify_rows")) return 1;
  sprout_launch(verify_decide_kernel, dim3(requests), dim3(THREADS), 0, stream, p);
  if (sprout_check_launch("verify_decide") || temperature == nullptr) return sprout_check_launch("verify_decide");
  // A launch less where the sums are one round of blocks on the device, half a block an SM where they have a draft's as well: calls of so
  // few wait for the host, beyond it the drawing block's work behind its sum takes longer than the launch.  Without draft logits, 3 and 4 launches:
  // 38 blocks 18.8 and 20.4 us a call, 228 18.9 and 21.0, 320 19.9 and 21.1, 342 22.9 and 21.2, 640 26.1 and 22.8; with them: 38 20.5 and
  // 21.3, 64 20.0 and 21.9, 76 21.8 and 21.6, 96 22.4 and 21.9, 256 27.6 and 26.4.
  const bool few = runs * requests * (draft_rows ? 4 : 1) <= 2 * sprout_sm_count();
  if (few) sprout_launch(verify_sums_kernel<true>, dim3((unsigned)(runs * requests)), dim3(THREADS), 0, stream, p);
  else sprout_launch(verify_sums_kernel<false>, dim3((unsigned)(runs * requests)), dim3(THREADS), 0, stream, p);
  if (sprout_check_launch("verify_sums") || few) return sprout_check_launch("verify_sums");
  sprout_launch(verify_draw_kernel, dim3(requests), dim3(DRAW_THREADS), 0, stream, p);
  return sprout_check_launch("verify_draw");
}
