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
// another: float32 exponentials leave the running sum off by 1e-8 and would pick the neighbour once in a few hundred draws.  So
// exponentials and sums are 64-bit (`pow2`: 1e-12).
//
// Two launches.  verify_rows_kernel: a block per (row, run of RUN logits) holds the run in registers: its maximum, first index,
// sum of exponentials.  verify_pick_kernel: a cluster of CTAs per request merges the runs of its rows, finds the first row that does
// not stand, and draws: where nothing is taken away from p, from the sums of the runs there are and one run's logits; else the CTAs add
// up max(p - q, 0) over a share of the runs each and exchange the sums, and the one in whose share the draw falls looks through it.
#include <cooperative_groups.h>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int THREADS = 256, PER_THREAD = 16, RUN = THREADS * PER_THREAD;     // logits of a run
constexpr int WARPS = THREADS / 32;
constexpr int CTAS = 8;                    // of a request's cluster

struct RunSum { double sum; float max; int index; int bad; int pad; };       // sum: of 2^((v - max) log2(e) / T)

// 2^y for y <= 0 to 1e-12: y = k + f with |f| <= 1/2, 2^f by a polynomial through the Chebyshev nodes, k into the exponent.
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
  return y < -1000.0 ? 0.0 : r;
}

__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ void better(float& v, int& i, float ov, int oi) {
  if (ov > v || (ov == v && oi < i)) { v = ov; i = oi; }
}

// The logit of a run that a thread's place i holds: side by side in fours over the threads, so that a warp reads whole lines, or
// (IN_ORDER) PER_THREAD side by side in every thread, for running sums.
template <bool IN_ORDER> __device__ __forceinline__ int place_of(int i) {
  return IN_ORDER ? (int)threadIdx.x * PER_THREAD + i : (i >> 2) * (THREADS * 4) + (int)threadIdx.x * 4 + (i & 3);
}
// PER_THREAD logits of a run of `count`; -inf beyond them.
template <bool IN_ORDER>
__device__ __forceinline__ void load_run(const float* run, int count, float (&v)[PER_THREAD]) {
  const bool aligned = ((uintptr_t)run & 15) == 0;
#pragma unroll
  for (int i = 0; i < PER_THREAD; i += 4) {
    const int at = place_of<IN_ORDER>(i);
    if (aligned && at + 4 <= count) {
      const float4 t = *(const float4*)(run + at);
      v[i] = t.x; v[i + 1] = t.y; v[i + 2] = t.z; v[i + 3] = t.w;
    } else {
#pragma unroll
      for (int k = 0; k < 4; k++) v[i + k] = at + k < count ? run[at + k] : -INFINITY;
    }
  }
}

struct Rows {
  const float* logits; const float* draft_logits;      // [rows, vocab], [draft_rows, vocab]
  long long ld, draft_ld;
  const int* row_start; const float* temperature;      // [requests + 1], [requests] (null: 0)
  RunSum* sums;                                        // [rows + draft_rows, runs]
  int rows, draft_rows, requests, vocab, runs;
};

__global__ void __launch_bounds__(THREADS)
verify_rows_kernel(const Rows p) {
  __shared__ float s_val[WARPS];
  __shared__ int s_idx[WARPS];
  __shared__ double s_sum[WARPS];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / p.runs, run = blockIdx.x % p.runs;
  const bool draft = row >= p.rows;
  const int own = draft ? row - p.rows : row;
  const float* base = draft ? p.draft_logits + (size_t)own * p.draft_ld : p.logits + (size_t)own * p.ld;
  // the row's request: the last whose rows (draft rows: one fewer per request before) begin at or before it
  int lo = 0, hi = p.requests - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (p.row_start[mid] - (draft ? mid : 0) <= own) lo = mid; else hi = mid - 1;
  }
  const float temp = p.temperature ? p.temperature[lo] : 0.f;
  if (draft && !(temp > 0.f)) return;                  // a greedy request's draft probabilities are not asked for
  const int begin = run * RUN, count = min(RUN, p.vocab - begin);
  float v[PER_THREAD];
  load_run<false>(base + begin, count, v);
  float best = -INFINITY;
  int best_i = 0x7fffffff, bad = 0;
#pragma unroll
  for (int i = 0; i < PER_THREAD; i++) {
    const int at = place_of<false>(i);
    if (at < count && !isfinite(v[i])) bad = 1;
    if (v[i] > best) { best = v[i]; best_i = begin + at; }         // places rise with i: the first maximum stays
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) better(best, best_i, __shfl_xor_sync(0xffffffffu, best, o), __shfl_xor_sync(0xffffffffu, best_i, o));
  if (lane == 0) { s_val[warp] = best; s_idx[warp] = best_i; }
  bad = __syncthreads_or(bad);
  best = s_val[0]; best_i = s_idx[0];
#pragma unroll
  for (int w = 1; w < WARPS; w++) better(best, best_i, s_val[w], s_idx[w]);
  double sum = 0.0;
  if (temp > 0.f && !bad) {
    const double c = 1.4426950408889634 / (double)temp, top = (double)best;
#pragma unroll
    for (int i = 0; i < PER_THREAD; i++) {
      const double e = pow2(((double)v[i] - top) * c);             // the difference first: it is exact next to the maximum, whatever T
      if (place_of<false>(i) < count) sum += e;
    }
    sum = warp_sum_d(sum);
    if (lane == 0) s_sum[warp] = sum;
    __syncthreads();
    sum = s_sum[0];
#pragma unroll
    for (int w = 1; w < WARPS; w++) sum += s_sum[w];
  }
  if (tid == 0) p.sums[(size_t)row * p.runs + run] = RunSum{sum, best, best_i, bad, 0};
}

struct Pick {
  Rows rows;
  const int* drafts; const float* accept; const float* draw;      // [rows]
  int* out; int* accepted; int* status;                           // [rows], [requests]
};

// What a row's runs add up to: its maximum, first index and (with `sums`) sum relative to the maximum, in every lane of the warp.
struct RowSum { double sum; float max; int index; int bad; };
__device__ __forceinline__ RowSum merge_runs(const RunSum* runs, int count, bool sums, double c) {
  const int lane = threadIdx.x & 31;
  float best = -INFINITY;
  int best_i = 0x7fffffff, bad = 0;
  for (int i = lane; i < count; i += 32) {
    better(best, best_i, runs[i].max, runs[i].index);
    bad |= runs[i].bad;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) better(best, best_i, __shfl_xor_sync(0xffffffffu, best, o), __shfl_xor_sync(0xffffffffu, best_i, o));
  bad = __any_sync(0xffffffffu, bad);
  double sum = 0.0;
  if (sums && !bad)
    for (int i = lane; i < count; i += 32) sum += runs[i].sum * pow2(((double)runs[i].max - (double)best) * c);
  return RowSum{warp_sum_d(sum), best, best_i, bad};
}

// The lowest place of a block's weights (PER_THREAD a thread, side by side) whose running sum, counted from `before`, exceeds `target`;
// the last with any weight where rounding left none.  -1 where nothing has weight.  `s_sum` [WARPS], `s_pick` [2] are shared.
__device__ __forceinline__ int pick_place(const double (&w)[PER_THREAD], double before, double target, double* s_sum, int* s_pick) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  double own = 0.0;
#pragma unroll
  for (int i = 0; i < PER_THREAD; i++) own += w[i];
  double upto = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double other = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += other;
  }
  __syncthreads();                                     // what these held has been read
  if (lane == 31) s_sum[warp] = upto;
  if (tid == 0) { s_pick[0] = 0x7fffffff; s_pick[1] = -1; }
  __syncthreads();
  double running = before;
  for (int i = 0; i < warp; i++) running += s_sum[i];
  running += upto - own;
  int first = 0x7fffffff, last = -1;
#pragma unroll
  for (int i = 0; i < PER_THREAD; i++) {
    running += w[i];
    if (w[i] > 0.0) {
      last = tid * PER_THREAD + i;
      if (running > target && first == 0x7fffffff) first = last;
    }
  }
  if (first != 0x7fffffff) atomicMin(&s_pick[0], first);
  if (last >= 0) atomicMax(&s_pick[1], last);
  __syncthreads();
  return s_pick[0] != 0x7fffffff ? s_pick[0] : s_pick[1];
}

__global__ void __cluster_dims__(CTAS, 1, 1) __launch_bounds__(THREADS)
verify_pick_kernel(const Pick p) {
  __shared__ double s_z[WARPS], s_zq[WARPS];
  __shared__ float s_m[WARPS], s_mq[WARPS];
  __shared__ int s_best[WARPS], s_code[WARPS];         // per row of a batch: 0 stands, 1 does not, 2 and more: flagged
  __shared__ double s_sum[WARPS], s_total[CTAS];
  __shared__ int s_pick[2], s_choice;
  __shared__ double s_before, s_target;
  pdl_launch_dependents();
  pdl_wait();
  const cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), r = blockIdx.x / CTAS;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Rows& a = p.rows;
  const int first = a.row_start[r], end = a.row_start[r + 1], count = end - first;
  // every CTA of the cluster takes the same decisions from the same numbers, up to where the cluster's CTAs part
  if (first < 0 || end > a.rows || count < 1 || (a.draft_rows > 0 && (first - r < 0 || end - r - 1 > a.draft_rows))) {
    if (rank == 0 && tid == 0) { atomicOr(p.status, SPROUT_STATUS_BAD_ROWS); p.accepted[r] = -1; }
    return;
  }
  const float temp = a.temperature ? a.temperature[r] : 0.f;
  const bool greedy = !(temp > 0.f);
  const double c = greedy ? 0.0 : 1.4426950408889634 / (double)temp;
  int row = 0, code = 0;
  for (int base = 0; base < count; base += WARPS) {
    const int i = base + warp;
    if (i < count) {
      const RowSum s = merge_runs(a.sums + (size_t)(first + i) * a.runs, a.runs, !greedy, c);
      int verdict = s.bad ? SPROUT_STATUS_NONFINITE : 1;           // the last row never "stands": the draw is made there
      double zq = 0.0;
      float mq = 0.f;
      if (i < count - 1 && !s.bad) {
        const int x = p.drafts[first + i];
        if (x < 0 || x >= a.vocab) {
          verdict = SPROUT_STATUS_BAD_TOKEN;
        } else if (greedy) {
          verdict = x == s.index ? 0 : 1;
        } else {
          const double px = pow2(((double)a.logits[(size_t)(first + i) * a.ld + x] - (double)s.max) * c) / s.sum;
          double qx = 1.0;
          if (a.draft_rows > 0) {
            const int d = first - r + i;
            const RowSum t = merge_runs(a.sums + (size_t)(a.rows + d) * a.runs, a.runs, !greedy, c);
            if (t.bad) verdict = SPROUT_STATUS_NONFINITE;
            zq = t.sum; mq = t.max;
            qx = pow2(((double)a.draft_logits[(size_t)d * a.draft_ld + x] - (double)mq) * c) / zq;
          }
          if (verdict == 1) verdict = (double)p.accept[first + i] * qx < px ? 0 : 1;
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
  if (rank == 0) {
    for (int i = tid; i < count; i += THREADS)
      if (i != row || code > 1) p.out[first + i] = i < row ? p.drafts[first + i] : -1;
    if (tid == 0) {
      p.accepted[r] = row;
      if (code > 1) atomicOr(p.status, code);
    }
  }
  if (code > 1) return;
  if (greedy) {
    if (rank == 0 && tid == 0) p.out[first + row] = s_best[slot];
    return;
  }
  const float* logits = a.logits + (size_t)(first + row) * a.ld;
  const float max_p = s_m[slot];
  const double z = s_z[slot], top = (double)max_p, draw = (double)p.draw[first + row];
  const bool take_away = row < count - 1;              // max(p - q, 0) instead of p
  double w[PER_THREAD];
  if (take_away && a.draft_rows > 0) {
    // the difference, over a share of the runs in every CTA
    const float* draft = a.draft_logits + (size_t)(first - r + row) * a.draft_ld;
    const double top_q = (double)s_mq[slot], inv_z = 1.0 / z, inv_zq = 1.0 / s_zq[slot];
    const int share = (a.runs + CTAS - 1) / CTAS, run0 = min(rank * share, a.runs), run1 = min(run0 + share, a.runs);
    auto difference = [&](int run) {
      float v[PER_THREAD], d[PER_THREAD];
      const int begin = run * RUN, n = min(RUN, a.vocab - begin);
      load_run<true>(logits + begin, n, v);
      load_run<true>(draft + begin, n, d);
      double sum = 0.0;
#pragma unroll
      for (int i = 0; i < PER_THREAD; i++) {
        const double e = pow2(((double)v[i] - top) * c) * inv_z - pow2(((double)d[i] - top_q) * c) * inv_zq;
        w[i] = tid * PER_THREAD + i < n ? fmax(e, 0.0) : 0.0;
        sum += w[i];
      }
      return sum;
    };
    auto block_total = [&](double sum) {
      sum = warp_sum_d(sum);
      __syncthreads();
      if (lane == 0) s_sum[warp] = sum;
      __syncthreads();
      sum = s_sum[0];
#pragma unroll
      for (int i = 1; i < WARPS; i++) sum += s_sum[i];
      return sum;
    };
    double mine = 0.0;
    for (int run = run0; run < run1; run++) mine += difference(run);
    mine = block_total(mine);
    cluster.sync();                                    // every CTA of the cluster runs: its shared memory may be written
    if (tid < CTAS) *cluster.map_shared_rank(&s_total[rank], tid) = mine;
    cluster.sync();
    double total = 0.0, before = 0.0;
    int owner = -1, last = -1;
    for (int i = 0; i < CTAS; i++) total += s_total[i];
    const double target = draw * total;
    double sum = 0.0;
    for (int i = 0; i < CTAS; i++) {
      if (s_total[i] > 0.0) last = i;
      if (owner < 0 && sum + s_total[i] > target) { owner = i; before = sum; }
      sum += s_total[i];
    }
    if (owner < 0 && last >= 0) {                      // rounding: the last share with any weight
      owner = last;
      before = 0.0;
      for (int i = 0; i < last; i++) before += s_total[i];
    }
    if (owner >= 0) {
      if (rank != owner) return;
      int chosen = -1;
      double at = before;
      bool falls = false;
      for (int run = run0; run < run1 && !falls; run++) {
        const double in_run = block_total(difference(run));
        if (!(in_run > 0.0)) continue;
        chosen = run;
        before = at;
        at += in_run;
        falls = at > target;
      }
      if (!falls) difference(chosen);                  // rounding: the last run with any weight
      const int place = pick_place(w, before, target, s_sum, s_pick);
      if (tid == 0) p.out[first + row] = chosen * RUN + place;
      return;
    }
    // p and q are the same everywhere (then nothing is rejected but by rounding): drawn from p
  }
  if (rank != 0) return;
  // from p, less the drafted token where it was rejected and nothing else was drafted with any probability
  const int without = take_away && a.draft_rows == 0 ? p.drafts[first + row] : -1;
  const RunSum* runs = a.sums + (size_t)(first + row) * a.runs;
  if (warp == 0) {
    // the runs' weights relative to the row's maximum, a lane each, in order
    auto weight = [&](int i, int skip) {
      if (i >= a.runs) return 0.0;
      double s = runs[i].sum;
      if (skip >= 0 && skip / RUN == i) s = fmax(0.0, s - pow2(((double)logits[skip] - (double)runs[i].max) * c));
      return s * pow2(((double)runs[i].max - top) * c);
    };
    auto sum_of = [&](int skip) {
      double s = 0.0;
      for (int i = lane; i < a.runs; i += 32) s += weight(i, skip);
      return warp_sum_d(s);
    };
    int skip = without;
    double total = sum_of(skip);
    if (!(total > 0.0)) {                              // the drafted token has all the weight there is: drawn from p
      skip = -1;
      total = z;
    }
    const double target = draw * total;
    double at = 0.0, before = 0.0;
    int chosen = -1;
    bool falls = false;
    for (int base = 0; base < a.runs && !falls; base += 32) {
      const double s = weight(base + lane, skip);
      double upto = s;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double other = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += other;
      }
      const unsigned any = __ballot_sync(0xffffffffu, s > 0.0), over = __ballot_sync(0xffffffffu, s > 0.0 && at + upto > target);
      if (any) {                                       // the first run that passes the target, or (so far) the last with any weight
        falls = over != 0;
        const int l = falls ? __ffs(over) - 1 : 31 - __clz(any);
        chosen = base + l;
        before = __shfl_sync(0xffffffffu, at + upto - s, l);
      }
      at += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane == 0) { s_choice = chosen; s_before = before; s_target = target; s_pick[0] = skip; }
  }
  __syncthreads();
  const int run = s_choice, skip = s_pick[0];
  __syncthreads();
  float v[PER_THREAD];
  const int begin = run * RUN, n = min(RUN, a.vocab - begin);
  load_run<true>(logits + begin, n, v);
#pragma unroll
  for (int i = 0; i < PER_THREAD; i++) {
    const int at = tid * PER_THREAD + i;
    w[i] = at < n && begin + at != skip ? pow2(((double)v[i] - top) * c) : 0.0;
  }
  const int place = pick_place(w, s_before, s_target, s_sum, s_pick);
  if (tid == 0) p.out[first + row] = place >= 0 ? begin + place : s_best[slot];
}

}  // namespace

// Bytes of scratch for `rows` rows (target's and draft's together) of `vocab` logits.
SPROUT_API long long sprout_verify_scratch_bytes(int rows, int vocab) { return (long long)rows * ((vocab + RUN - 1) / RUN) * (long long)sizeof(RunSum); }

// Request r's rows are row_start[r] .. row_start[r + 1] - 1 of `logits` [rows, vocab], at least one; its draft rows, one fewer, begin at
// row_start[r] - r of `draft_logits` (null with draft_rows 0: the drafts have no distribution).  temperature, accept and draw may be null
// together (all requests greedy).  Row i of `drafts` is the token drafted after row i's place; a request's last is not read.
SPROUT_API int sprout_verify(const float* logits, long long ld, const float* draft_logits, long long draft_ld, const int* drafts, const int* row_start,
                             const float* temperature, const float* accept, const float* draw, int* out, int* accepted, void* scratch,
                             int rows, int draft_rows, int requests, int vocab, int* status, cudaStream_t stream) {
  SPROUT_REQUIRE(rows > 0 && requests > 0 && requests <= rows && vocab > 0 && ld >= 0, "verify: bad sizes rows=%d requests=%d vocab=%d ld=%lld", rows, requests, vocab, ld);
  SPROUT_REQUIRE(draft_rows == 0 || (draft_rows == rows - requests && draft_logits && draft_ld >= 0), "verify: a draft row per drafted token");
  SPROUT_REQUIRE(logits && drafts && row_start && out && accepted && scratch && status, "verify: null pointer");
  SPROUT_REQUIRE((temperature == nullptr) == (accept == nullptr) && (accept == nullptr) == (draw == nullptr), "verify: temperatures and both kinds of uniform numbers go together");
  const int runs = (vocab + RUN - 1) / RUN;
  SPROUT_REQUIRE((long long)runs * (rows + (long long)draft_rows) <= 0x7fffffffLL && (long long)requests * CTAS <= 0x7fffffffLL, "verify: too many rows");
  Pick p;
  p.rows = Rows{logits, draft_logits, ld, draft_ld, row_start, temperature, (RunSum*)scratch, rows, draft_rows, requests, vocab, runs};
  p.drafts = drafts; p.accept = accept; p.draw = draw; p.out = out; p.accepted = accepted; p.status = status;
  sprout_launch(verify_rows_kernel, dim3(runs * (rows + draft_rows)), dim3(THREADS), 0, stream, p.rows);
  if (sprout_check_launch("verify_rows")) return 1;
  sprout_launch(verify_pick_kernel, dim3(requests * CTAS), dim3(THREADS), 0, stream, p);
  return sprout_check_launch("verify_pick");
}
