// Losses over the tokens of many sequences, and their gradients: the clipped policy loss with KL and entropy terms, and the
// preference loss of paired sequences.
//
// Tokens lie in one array; sequence s has those from offsets[s] to offsets[s + 1], or every sequence `length` of them, and of
// these the ones whose mask byte is not 0 count.  What is summed over a sequence (how many count, their log-ratios, the terms of
// the loss) is summed in three steps, in an order that depends on the sizes alone:
//   parts    a wave takes a chunk of tokens, whatever sequences they are of, and leaves the sums of each of them: chunk c and
//            sequence s share the place c + s, and no other pair does, since one of the two grows from pair to pair.  Long and short
//            sequences are the same work here and in the gradient, and nothing has to be cleared.
//   join     every sequence's parts are added up by as many lanes as a sequence has parts on average, the loss formed, and what a
//            token's gradient needs of its sequence.  One long sequence among short ones waits for its few lanes: 1024 sequences of
//            4.2 million tokens take 38 us forward when they are equal and 289 when one of them holds nine tenths; 16 of 147 456
//            16.1 and 17.6.
//   gradient tokens as they lie (backward)
// Up to 100 000 tokens bound by the latency of two launches forward (7 to 17 us in a graph) and one backward (2 to 4), so that a wave
// has a single row of 64 tokens until there are enough for every CU; 4.2 million tokens with everything that there is (89 MB) take 35 and
// 21 us, a sixth of it exponentials.  Terms are formed in float64: a ratio's side of a clipping border decides about its whole
// gradient, and the KL estimators are differences of nearly equal numbers.
#include "mx_rows.h"

namespace mx {

constexpr int kSeqGrad = 256;          // lanes of a workgroup of the gradient
constexpr int kSeqFew = 1024;          // lanes of the workgroup that joins alone
constexpr int kSeqMany = 256;          // lanes of a workgroup where several join
constexpr int kSeqManyGroups = 1024;   // of which there are at most
// Tokens from which on a wave takes 4 rows of 64 (us forward in a graph, 1 / 4 rows.  Below: 16 sequences of 61 10.0 / 15.9, 16 of 1024 9.7 /
// 11.3, 64 of 400 11.6 / 12.4, 64 of 511 11.9 / 12.5, one of 30 000 12.0 / 11.8.  From there on: one of 34 000 11.6 / 12.1, 64 of 600 13.6 /
// 12.5, 16 of 4096 14.0 / 11.8, one of 147 456 20.7 / 13.9, 1024 of 4099 46.9 / 37.7, 8 rows 43.0 there, 16 63.6.  Short sequences
// would want single rows for longer: 512 of 70 11.4 / 16.6), and in the gradient (us, 1 / 4 rows, packed: 128 sequences of 4099 6.0 /
// 7.4, 1024 of 4099 30.8 / 24.5).
constexpr int64_t kSeqLong = 32768, kSeqGradLong = 1 << 20;
__host__ __device__ __forceinline__ int seq_rows(int64_t tokens) { return tokens < kSeqLong ? 1 : 4; }
__host__ __device__ __forceinline__ int64_t seq_chunks(int64_t tokens) {
  const int64_t chunk = 64 * seq_rows(tokens);
  return (tokens + chunk - 1) / chunk;
}

// Log-probabilities, bf16 or float32
struct SeqValues {
  const void* p;
  int f32;
  __device__ __forceinline__ float at(int64_t i) const {
    return f32 ? ((const float*)p)[i] : bf16_lo(((const uint16_t*)p)[i]);
  }
};

struct Sequences {
  const void* offsets;  // [count + 1], or null: `length` tokens each
  int64_t count, tokens, length;
  const uint8_t* mask;  // or null
  int wide;             // offsets are int64
  // (offsets outside the array, or that fall, are not followed out of it)
  __device__ __forceinline__ int64_t offset(int64_t s) const {
    if (!offsets) return s * length;
    const int64_t at = wide ? ((const int64_t*)offsets)[s] : (int64_t)((const int32_t*)offsets)[s];
    return at < 0 ? 0 : at > tokens ? tokens : at;
  }
  // The sequence of token i < tokens, from `first` on: -1 before the first one, `count` behind the last.
  __device__ __forceinline__ int64_t find(int64_t i, int64_t first = -1) const {
    if (!offsets) return (uint32_t)i / (uint32_t)length;  // (tokens and the row behind them fit 32 bits)
    int64_t lo = first, hi = count + 1;  // the last place whose offset is not behind i
    while (hi - lo > 1) {
      const int64_t mid = (lo + hi) >> 1;
      if (offset(mid) <= i) lo = mid; else hi = mid;
    }
    return lo;
  }
};

// The same for a whole wave with one token i: its lanes look at 64 offsets at a time, two or three rounds where a search by halves
// takes ten that wait for each other (us forward and backward with those and without: 1024 packed sequences of 4099 43.3 and 30.9, 41.0 and
// 24.7; 32 768 of 128 69 and 64, 51 and 31).
__device__ __forceinline__ int64_t seq_find(const Sequences& q, int64_t i, int lane) {
  if (!q.offsets) return q.find(i);
  int64_t lo = -1, hi = q.count + 1;
  while (hi - lo > 1) {
    const int64_t step = (hi - lo - 1 + 63) / 64, at = lo + (lane + 1) * step;
    const int64_t below = __popcll(__ballot(at < hi && q.offset(at) <= i));
    hi = below < 64 && lo + (below + 1) * step < hi ? lo + (below + 1) * step : hi;
    lo += below * step;
  }
  return lo;
}
// The sequence of each lane's token in the row from `row` on, whose first token is of sequence s or a later one.
__device__ __forceinline__ int64_t seq_of_row(const Sequences& q, int64_t s, int64_t row, int lane) {
  if (!q.offsets) return q.find(row + lane);
  const int64_t next = s + 1 + lane <= q.count ? q.offset(s + 1 + lane) : INT64_MAX;
  const int ends = __popcll(__ballot(next <= row + 63));
  if (ends > 8) return q.find(row + lane, s);
  int64_t mine = s;
  for (int j = 0; j < ends; ++j) mine += row + lane >= __shfl(next, j, 64);
  return mine;
}

struct Policy {
  SeqValues lp, old, ref;  // p null: none
  const float* advantages;
  int advantage_tokens;    // one for every token, else for every sequence
  int whole;               // one ratio a sequence
  int by_sequence;         // means over sequences of means over their tokens, else over all tokens
  int kl;                  // 0 k1, 1 k2, 2 k3, 3 k3 swapped
  double low, high;        // the ratio's borders
  double kl_coef, entropy_coef;
};
struct Preference {
  SeqValues lp, ref;
  int kind;  // 0 sigmoid, 1 hinge, 2 squared
  int mean;  // means of log-ratios, else sums
  double beta, smoothing;
};

// -min(r A, clip(r) A): for A >= 0 the smaller, for A < 0 the larger of r and its border (0 where A is 0, whatever r is)
__device__ __forceinline__ double seq_objective(const Policy& f, double r, double A) {
  return A >= 0 ? -A * (r > f.high ? f.high : r) : -A * (r < f.low ? f.low : r);
}
__device__ __forceinline__ bool seq_clipped(const Policy& f, double r) {
  const double c = r > f.high ? f.high : r < f.low ? f.low : r;
  return fabs(r - c) > 1e-6;
}
// e^x, e^x - 1 and e^x - 1 - x (infinite where x is) to 1e-14 of each: x = k ln 2 + t, |t| <= ln 2 / 2, and
// e^t - 1 - t = t^2 (1/2! + t/3! + ...) up to t^12 / 12!.
struct SeqExp {
  double e, minus, rest;
};
__device__ __forceinline__ SeqExp seq_exp(double x) {
  const double bounded = x > 750.0 ? 750.0 : x < -750.0 ? -750.0 : x;  // (NaN stays)
  const double k = __builtin_rint(bounded * 1.4426950408889634);
  const double t = __builtin_fma(-k, 2.3190468138462996e-17, __builtin_fma(-k, 0.6931471805599453, bounded));
  double q = 1.0 / 479001600;
  constexpr double kBelow[10] = {1.0 / 39916800, 1.0 / 3628800, 1.0 / 362880, 1.0 / 40320, 1.0 / 5040,
                                 1.0 / 720,      1.0 / 120,     1.0 / 24,     1.0 / 6,     1.0 / 2};
#pragma unroll
  for (int n = 0; n < 10; ++n) q = __builtin_fma(q, t, kBelow[n]);
  const double rest = t * t * q, minus = t + rest;
  const double e = ldexp(1.0 + minus, (int)k);
  return k == 0.0 ? SeqExp{e, minus, rest} : SeqExp{e, e - 1.0, x > 750.0 ? e : e - 1.0 - x};
}
__device__ __forceinline__ double seq_kl(int kind, double x) {
  if (kind == 0) return x;
  if (kind == 1) return 0.5 * x * x;
  return seq_exp(kind == 2 ? -x : x).rest;
}
__device__ __forceinline__ double seq_kl_slope(int kind, double x) {
  if (kind == 0) return 1.0;
  if (kind == 1) return x;
  const double minus = seq_exp(kind == 2 ? -x : x).minus;
  return kind == 2 ? -minus : minus;
}

// Sums over a wave, in every lane: 16 lanes by moves between lanes, then two steps through the LDS crossbar.
template <int CTRL>
__device__ __forceinline__ double seq_moved(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, (uint64_t)dpp<CTRL>((uint32_t)b) | (uint64_t)dpp<CTRL>((uint32_t)(b >> 32)) << 32);
}
__device__ __forceinline__ double seq_wave_sum(double v) {
  v += seq_moved<kQuadXor1>(v);
  v += seq_moved<kQuadXor2>(v);
  v += seq_moved<kRowHalfMirror>(v);
  v += seq_moved<kRowMirror>(v);
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

// What is read of a token, and what it adds to its sequence's sums.
struct SeqToken {
  float lp, old, ref, advantage;
  bool counts;
};
constexpr int kPolicySums = 7;      // tokens, x, lp, kl, objective, ratio, clipped
constexpr int kPreferenceSums = 2;  // tokens, x

__device__ __forceinline__ SeqToken seq_load(const Policy& f, const Sequences& q, int64_t i) {
  SeqToken t = {0.f, 0.f, 0.f, 0.f, i < q.tokens};
  if (t.counts) {
    t.lp = f.lp.at(i);
    if (f.old.p) t.old = f.old.at(i);
    if (f.ref.p) t.ref = f.ref.at(i);
    if (f.advantage_tokens) t.advantage = f.advantages[i];
    if (q.mask) t.counts = q.mask[i] != 0;
  }
  return t;
}
__device__ __forceinline__ SeqToken seq_load(const Preference& f, const Sequences& q, int64_t i) {
  SeqToken t = {0.f, 0.f, 0.f, 0.f, i < q.tokens};
  if (t.counts) {
    t.lp = f.lp.at(i);
    if (f.ref.p) t.ref = f.ref.at(i);
    if (q.mask) t.counts = q.mask[i] != 0;
  }
  return t;
}
__device__ __forceinline__ double seq_advantage(const Policy& f, const SeqToken& t, int64_t s) {
  return (double)(f.advantage_tokens ? t.advantage : f.advantages[s]);
}
__device__ __forceinline__ void seq_add(const Policy& f, const SeqToken& t, int64_t s, double (&sum)[kPolicySums]) {
  const double lp = (double)t.lp, x = f.old.p ? lp - (double)t.old : 0.0;
  sum[0] += 1.0;
  sum[1] += x;
  sum[2] += lp;
  if (f.ref.p) sum[3] += seq_kl(f.kl, lp - (double)t.ref);
  if (!f.whole) {
    const double r = seq_exp(x).e;
    sum[4] += seq_objective(f, r, seq_advantage(f, t, s));
    sum[5] += r;
    sum[6] += seq_clipped(f, r) ? 1.0 : 0.0;
  }
}
__device__ __forceinline__ void seq_add(const Preference& f, const SeqToken& t, int64_t, double (&sum)[kPreferenceSums]) {
  sum[0] += 1.0;
  sum[1] += f.ref.p ? (double)t.lp - (double)t.ref : (double)t.lp;
}

// parts: [chunks + count][SUMS].  A wave's chunk is ROWS rows of 64 tokens.  Rows inside one sequence are added up lane by lane; in a row
// that sequences end in, those that lie in it whole are summed among their lanes, and the running one is summed up and left.
template <int SUMS, int ROWS, class F>
__device__ __forceinline__ void seq_parts(const F& f, const Sequences& q, int64_t chunk, int lane, double* parts) {
  constexpr int kChunk = 64 * ROWS;
  const int64_t begin = chunk * kChunk, end = begin + kChunk < q.tokens ? begin + kChunk : q.tokens;
  SeqToken t[ROWS];
#pragma unroll
  for (int k = 0; k < ROWS; ++k) t[k] = seq_load(f, q, begin + k * 64 + lane);
  int64_t s = seq_find(q, begin, lane);
  int64_t stop = s < 0 || s >= q.count ? begin : q.offset(s + 1);
  double sum[SUMS];
  auto clear = [&]() {
#pragma unroll
    for (int k = 0; k < SUMS; ++k) sum[k] = 0.0;
  };
  auto leave = [&]() {  // the running sequence's sums
    if (s < 0 || s >= q.count) return;
#pragma unroll
    for (int k = 0; k < SUMS; ++k) {
      const double all = seq_wave_sum(sum[k]);
      if (lane == k) parts[(chunk + s) * SUMS + k] = all;
    }
  };
  clear();
#pragma unroll
  for (int k = 0; k < ROWS; ++k) {
    const int64_t row = begin + k * 64, i = row + lane;
    if (row >= end) break;
    if (stop >= (row + 64 < end ? row + 64 : end)) {
      if (t[k].counts) seq_add(f, t[k], s, sum);
      continue;
    }
    const int64_t of = seq_of_row(q, s, row, lane), mine = i < end ? of : q.count;
    double v[SUMS];
#pragma unroll
    for (int j = 0; j < SUMS; ++j) v[j] = 0.0;
    if (mine >= 0 && mine < q.count && t[k].counts) seq_add(f, t[k], mine, v);
    if (mine == s)
#pragma unroll
      for (int j = 0; j < SUMS; ++j) sum[j] += v[j];
    const int64_t last = __shfl(mine, 63, 64);
    if (last == s) continue;
    leave();
    const bool middle = mine != s && mine != last;
#pragma unroll
    for (int j = 0; j < SUMS; ++j) sum[j] = mine == last ? v[j] : 0.0;
    if (__ballot(middle)) {
      for (int off = 1; off < 64; off <<= 1) {
        const int64_t other = __shfl_down(mine, off, 64);
        const bool same = lane + off < 64 && other == mine;
#pragma unroll
        for (int j = 0; j < SUMS; ++j) {
          const double more = __shfl_down(v[j], off, 64);
          if (same) v[j] += more;
        }
      }
      const int64_t before = __shfl_up(mine, 1, 64);
      if (middle && mine >= 0 && mine < q.count && (lane == 0 || before != mine))
#pragma unroll
        for (int j = 0; j < SUMS; ++j) parts[(chunk + mine) * SUMS + j] = v[j];
    }
    s = last;
    stop = s < 0 || s >= q.count ? row : q.offset(s + 1);
  }
  leave();
}

template <int SUMS, int ROWS, class F>
__global__ __launch_bounds__(64) void seq_parts_kernel(F f, Sequences q, double* __restrict__ parts) {
  seq_parts<SUMS, ROWS>(f, q, blockIdx.x, threadIdx.x, parts);
}

// The sums of sequence s from its parts, in the first of `lanes` lanes that take them in turn (others: part of them).
template <int SUMS>
__device__ __forceinline__ void seq_joined(const Sequences& q, const double* parts, int64_t s, int lane, int lanes,
                                           double (&sum)[SUMS]) {
#pragma unroll
  for (int k = 0; k < SUMS; ++k) sum[k] = 0.0;
  const int64_t begin = q.offset(s), end = q.offset(s + 1);
  const int chunk = seq_rows(q.tokens) == 1 ? 6 : 8;  // (tokens of a chunk, as a power of two)
  if (end > begin) {
    const int64_t last = (end - 1) >> chunk;
#pragma unroll 4
    for (int64_t c = (begin >> chunk) + lane; c <= last; c += lanes)
#pragma unroll
      for (int k = 0; k < SUMS; ++k) sum[k] += parts[(c + s) * SUMS + k];
  }
  for (int off = 1; off < lanes; off <<= 1)
#pragma unroll
    for (int k = 0; k < SUMS; ++k) sum[k] += __shfl_xor(sum[k], off, 64);
}

// Sums over the lanes of the workgroup, in lane 0.
template <int LANES, int N>
__device__ __forceinline__ void seq_group_sum(double (&v)[N]) {
  constexpr int kWaves = LANES / 64;
  __shared__ double shared[kWaves][N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    v[k] = seq_wave_sum(v[k]);
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6][k] = v[k];
  }
  __syncthreads();
  if (threadIdx.x >= 64) return;
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = seq_wave_sum(threadIdx.x < kWaves ? shared[threadIdx.x][k] : 0.0);
}

// Sums over all sequences.  Policy: tokens, sequences that have some; by token objective, kl, ratio, clipped; by sequence the
// same; lp.  Preference: losses, pairs.
constexpr int kPolicyTotals = 11, kPreferenceTotals = 2;

// Of the sequence: for the gradient, each[2 s] tokens, each[2 s + 1] what its ratio adds to a token's gradient.
__device__ __forceinline__ void seq_take(const Policy& f, const Sequences& q, const double* parts, int64_t s, int lane,
                                         int lanes, double* __restrict__ each, float*, double (&total)[kPolicyTotals]) {
  double sum[kPolicySums];
  seq_joined(q, parts, s, lane, lanes, sum);
  if (lane) return;
  const double n = sum[0];
  double slope = 0.0;
  if (n > 0.0) {
    if (f.whole) {
      const double r = seq_exp(sum[1] / n).e, A = (double)f.advantages[s];
      if (A >= 0 ? !(r > f.high) : !(r < f.low)) slope = -A * r;
      sum[4] = n * seq_objective(f, r, A);
      sum[5] = n * r;
      sum[6] = seq_clipped(f, r) ? n : 0.0;
    }
    total[0] += n;
    total[1] += 1.0;
    total[2] += sum[4], total[3] += sum[3], total[4] += sum[5], total[5] += sum[6];
    total[6] += sum[4] / n, total[7] += sum[3] / n, total[8] += sum[5] / n, total[9] += sum[6] / n;
    total[10] += sum[2];
  }
  if (each) each[2 * s] = n, each[2 * s + 1] = slope;
}
__device__ __forceinline__ void seq_finish(const Policy& f, const Sequences& q, const double (&total)[kPolicyTotals],
                                           double* __restrict__ each, float* __restrict__ loss, float* __restrict__ metrics) {
  const double tokens = total[0] > 0 ? total[0] : 1.0, filled = total[1] > 0 ? total[1] : 1.0;
  const double pg = f.by_sequence ? total[6] / filled : total[2] / tokens, kl = f.by_sequence ? total[7] / filled : total[3] / tokens;
  const double entropy = -total[10] / tokens;
  // (a coefficient of 0 leaves out a term that is no number, too)
  *loss = (float)(pg + (f.kl_coef != 0 ? f.kl_coef * kl : 0.0) - (f.entropy_coef != 0 ? f.entropy_coef * entropy : 0.0));
  metrics[0] = (float)pg;
  metrics[1] = (float)kl;
  metrics[2] = (float)entropy;
  metrics[3] = (float)(f.whole ? total[8] / filled : total[4] / tokens);
  metrics[4] = (float)(f.whole ? total[9] / filled : total[5] / tokens);
  if (each) each[2 * q.count] = tokens, each[2 * q.count + 1] = filled;
}

// Of the pair: for the gradient, each[s] that of a token of either sequence (but for the mean over the pairs).  A sequence without
// tokens beside one that has some has h = 0.
__device__ __forceinline__ void seq_take(const Preference& f, const Sequences& q, const double* parts, int64_t p, int lane,
                                         int lanes, double* __restrict__ each, float* __restrict__ rewards,
                                         double (&total)[kPreferenceTotals]) {
  const int64_t other = q.count / 2 + p;
  double one[kPreferenceSums], two[kPreferenceSums];
  seq_joined(q, parts, p, lane, lanes, one);
  seq_joined(q, parts, other, lane, lanes, two);
  if (lane) return;
  const double of1 = f.mean && one[0] > 0 ? 1.0 / one[0] : 1.0, of2 = f.mean && two[0] > 0 ? 1.0 / two[0] : 1.0;
  const double h1 = one[1] * of1, h2 = two[1] * of2, z = h1 - h2, y = f.beta * z;
  double value, slope;
  if (f.kind == 0) {
    // -log sigmoid(y) = log(1 + e^-|y|) + max(-y, 0), and the sigmoids of y and -y from the same e^-|y|
    const double e = seq_exp(-fabs(y)).e, both = log1p(e), large = 1.0 / (1.0 + e), small = e * large;
    value = both + (y < 0 ? (1.0 - f.smoothing) * -y : f.smoothing != 0 ? f.smoothing * y : 0.0);  // (no part of an infinite y)
    slope = f.beta * (y < 0 ? f.smoothing * small - (1.0 - f.smoothing) * large : f.smoothing * large - (1.0 - f.smoothing) * small);
  } else if (f.kind == 1) {
    value = 1.0 - y < 0 ? 0.0 : 1.0 - y;  // (NaN stays)
    slope = y < 1.0 ? -f.beta : 0.0;
  } else {
    const double left = z - 0.5 / f.beta;
    value = left * left;
    slope = 2.0 * left;
  }
  if (one[0] + two[0] > 0) total[0] += value, total[1] += 1.0;
  rewards[p] = (float)(f.beta * h1);
  rewards[other] = (float)(f.beta * h2);
  if (each) each[p] = slope * of1, each[other] = -slope * of2;
}
__device__ __forceinline__ void seq_finish(const Preference&, const Sequences& q, const double (&total)[kPreferenceTotals],
                                           double* __restrict__ each, float* __restrict__ loss, float*) {
  const double pairs = total[1] > 0 ? total[1] : 1.0;
  *loss = (float)(total[0] / pairs);
  if (each) each[q.count] = pairs;
}

template <class F> struct SeqOf;
template <> struct SeqOf<Policy> { static constexpr int kSums = kPolicySums, kTotals = kPolicyTotals; };
template <> struct SeqOf<Preference> { static constexpr int kSums = kPreferenceSums, kTotals = kPreferenceTotals; };

// `lanes` lanes a sequence (or pair), `items` of them.  One workgroup finishes the loss; several leave their sums in `totals`.
template <int LANES, class F>
__device__ __forceinline__ void seq_join(const F& f, const Sequences& q, int64_t items, int lanes, const double* parts, double* totals,
                                         double* __restrict__ each, float* __restrict__ loss, float* __restrict__ more) {
  constexpr int kTotals = SeqOf<F>::kTotals;
  double total[kTotals];
#pragma unroll
  for (int k = 0; k < kTotals; ++k) total[k] = 0.0;
  const int lane = threadIdx.x & (lanes - 1), groups = LANES / lanes;
  for (int64_t s = (int64_t)blockIdx.x * groups + threadIdx.x / lanes; s < items; s += (int64_t)gridDim.x * groups)
    seq_take(f, q, parts, s, lane, lanes, each, more, total);
  seq_group_sum<LANES>(total);
  if (threadIdx.x == 0) {
    if (gridDim.x == 1) {
      seq_finish(f, q, total, each, loss, more);
    } else {
#pragma unroll
      for (int k = 0; k < kTotals; ++k) totals[(int64_t)blockIdx.x * kTotals + k] = total[k];
    }
  }
}
template <int LANES, class F>
__global__ __launch_bounds__(LANES) void seq_join_kernel(F f, Sequences q, int64_t items, int lanes, const double* __restrict__ parts,
                                                         double* __restrict__ totals, double* __restrict__ each,
                                                         float* __restrict__ loss, float* __restrict__ more) {
  seq_join<LANES>(f, q, items, lanes, parts, totals, each, loss, more);
}
template <class F>
__global__ __launch_bounds__(kSeqMany) void seq_finish_kernel(F f, Sequences q, int groups, const double* __restrict__ totals,
                                                              double* __restrict__ each, float* __restrict__ loss,
                                                              float* __restrict__ more) {
  constexpr int kTotals = SeqOf<F>::kTotals;
  double total[kTotals];
#pragma unroll
  for (int k = 0; k < kTotals; ++k) total[k] = 0.0;
  for (int g = threadIdx.x; g < groups; g += kSeqMany)
#pragma unroll
    for (int k = 0; k < kTotals; ++k) total[k] += totals[(int64_t)g * kTotals + k];
  seq_group_sum<kSeqMany>(total);
  if (threadIdx.x == 0) seq_finish(f, q, total, each, loss, more);
}
// The gradient of one token that counts.
__device__ __forceinline__ double seq_grad(const Policy& f, double share, double entropy, double slope, const SeqToken& t, int64_t s) {
  const double lp = (double)t.lp;
  double g = slope;
  if (!f.whole) {
    const double r = f.old.p ? seq_exp(lp - (double)t.old).e : 1.0, A = seq_advantage(f, t, s);
    if (A >= 0 ? !(r > f.high) : !(r < f.low)) g = -A * r;
  }
  if (f.ref.p && f.kl_coef != 0.0) g += f.kl_coef * seq_kl_slope(f.kl, lp - (double)t.ref);
  return g * share + entropy;
}
__device__ __forceinline__ double seq_grad(const Preference&, double share, double, double slope, const SeqToken&, int64_t) {
  return slope * share;
}
// What the tokens of sequence s have in common: the share of each in the means, the entropy's gradient, what the sequence adds.
__device__ __forceinline__ void seq_common(const Policy& f, const double* __restrict__ each, int64_t count, int64_t s, double& share,
                                           double& entropy, double& slope) {
  const double tokens = 1.0 / each[2 * count];
  share = f.by_sequence ? 1.0 / (each[2 * count + 1] * each[2 * s]) : tokens;
  entropy = f.entropy_coef * tokens;
  slope = each[2 * s + 1];
}
__device__ __forceinline__ void seq_common(const Preference&, const double* __restrict__ each, int64_t count, int64_t s, double& share,
                                           double&, double& slope) {
  share = 1.0 / each[count];
  slope = each[s];
}

// grad[i] = dloss * (that, where token i counts, else 0)
template <int ROWS, class F>
__global__ __launch_bounds__(kSeqGrad) void seq_grad_kernel(F f, Sequences q, const double* __restrict__ each,
                                                            const float* __restrict__ dloss, void* __restrict__ grad) {
  const int64_t begin = ((int64_t)blockIdx.x * (kSeqGrad / 64) + (threadIdx.x >> 6)) * (64 * ROWS);
  const int lane = threadIdx.x & 63;
  if (begin >= q.tokens) return;
  SeqToken t[ROWS];
#pragma unroll
  for (int k = 0; k < ROWS; ++k) t[k] = seq_load(f, q, begin + k * 64 + lane);
  const double by = (double)*dloss;
  const int64_t first = seq_find(q, begin, lane), end = begin + 64 * ROWS < q.tokens ? begin + 64 * ROWS : q.tokens;
  const bool one = first >= 0 && first < q.count && q.offset(first + 1) >= end;  // all of one sequence
  double share = 0.0, entropy = 0.0, slope = 0.0;
  if (one) seq_common(f, each, q.count, first, share, entropy, slope);
  int64_t s = first;
#pragma unroll
  for (int k = 0; k < ROWS; ++k) {
    const int64_t row = begin + k * 64, i = row + lane;
    if (row >= q.tokens) break;
    if (!one) s = seq_of_row(q, s, row, lane);
    double g = 0.0;
    if (t[k].counts && s >= 0 && s < q.count) {
      if (!one) seq_common(f, each, q.count, s, share, entropy, slope);
      g = seq_grad(f, share, entropy, slope, t[k], s) * by;
    }
    if (!one) s = __shfl(s, 63, 64);
    if (i >= q.tokens) continue;
    if (f.lp.f32) ((float*)grad)[i] = (float)g;
    else ((uint16_t*)grad)[i] = (uint16_t)__builtin_bit_cast(uint32_t, __builtin_convertvector(v2f_t{(float)g, 0.f}, v2bf_t));
  }
}

static int seq_check(const Sequences& q) {
  if (q.count < 0 || q.tokens < 0 || (q.count == 0 && !q.offsets && q.tokens > 0)) return MX_ERR_INVALID_ARG;
  if (!q.offsets && (q.length < 0 || (q.length ? q.tokens % q.length || q.tokens / q.length != q.count : q.tokens > 0)))
    return MX_ERR_INVALID_ARG;
  if ((uintptr_t)q.offsets & (q.wide ? 7 : 3)) return MX_ERR_ALIGNMENT;
  // (a wave for every chunk, a lane for every token: launches have fewer than 2^32 lanes)
  if (q.tokens > 0xFFFFFF00 || q.count > 0x3FFFFFFF) return MX_ERR_UNSUPPORTED;
  return MX_OK;
}
static bool seq_odd(const SeqValues& v) { return (uintptr_t)v.p & (v.f32 ? 3 : 1); }

// Lanes that add up a sequence's parts: about as many as it has of them on average.
static int seq_lanes(const Sequences& q) {
  const int64_t each = q.count ? seq_chunks(q.tokens) / q.count : 0;
  int lanes = 1;
  while (lanes < 64 && lanes < each) lanes *= 2;
  return lanes;
}

// Two launches, or three where one workgroup would have more than two rounds of sequences to join (four rounds of 512 packed pairs 19 us;
// by several workgroups and one that finishes 6 and 4).  (One workgroup for parts and join of few tokens: 976 of 16 sequences 11.4 us
// forward, in two launches 10.1.)
template <class F>
static void seq_loss(const F& f, const Sequences& q, int64_t items, double* parts, double* each, float* loss, float* more,
                     hipStream_t st) {
  constexpr int kSums = SeqOf<F>::kSums;
  const int64_t chunks = seq_chunks(q.tokens);
  const int lanes = seq_lanes(q);
  const bool alone = items * lanes <= 2 * kSeqFew;
  if (chunks) {
    if (seq_rows(q.tokens) == 1) hipLaunchKernelGGL((seq_parts_kernel<kSums, 1, F>), dim3((unsigned)chunks), dim3(64), 0, st, f, q, parts);
    else hipLaunchKernelGGL((seq_parts_kernel<kSums, 4, F>), dim3((unsigned)chunks), dim3(64), 0, st, f, q, parts);
  }
  if (alone) {
    hipLaunchKernelGGL((seq_join_kernel<kSeqFew, F>), dim3(1), dim3(kSeqFew), 0, st, f, q, items, lanes, (const double*)parts,
                       (double*)nullptr, each, loss, more);
    return;
  }
  const int64_t rounds = (items * lanes + kSeqMany - 1) / kSeqMany;
  const int groups = rounds < kSeqManyGroups ? (int)rounds : kSeqManyGroups;
  double* const totals = parts + (chunks + q.count) * kSums;
  hipLaunchKernelGGL((seq_join_kernel<kSeqMany, F>), dim3(groups), dim3(kSeqMany), 0, st, f, q, items, lanes, (const double*)parts,
                     totals, each, loss, more);
  hipLaunchKernelGGL(seq_finish_kernel<F>, dim3(1), dim3(kSeqMany), 0, st, f, q, groups, (const double*)totals, each, loss, more);
}
template <class F>
static void seq_grads(const F& f, const Sequences& q, const double* each, const float* dloss, void* grad, hipStream_t st) {
  const int rows = q.tokens < kSeqGradLong ? 1 : 4;
  const int64_t per = kSeqGrad * rows;
  const dim3 grid((unsigned)((q.tokens + per - 1) / per));
  if (rows == 1) hipLaunchKernelGGL((seq_grad_kernel<1, F>), grid, dim3(kSeqGrad), 0, st, f, q, each, dloss, grad);
  else hipLaunchKernelGGL((seq_grad_kernel<4, F>), grid, dim3(kSeqGrad), 0, st, f, q, each, dloss, grad);
}

static int status() { return hipGetLastError() == hipSuccess ? MX_OK : MX_ERR_LAUNCH; }

}  // namespace mx

using namespace mx;

extern "C" int64_t mx_sequence_loss_workspace(int64_t tokens, int64_t sequences) {
  if (tokens < 0 || sequences < 0) return 0;
  return 8 * (kPolicySums * (seq_chunks(tokens) + sequences) + kPolicyTotals * kSeqManyGroups);
}

static int policy_check(const mx_policy_loss_t* a, Policy& f, Sequences& q) {
  if (!a) return MX_ERR_INVALID_ARG;
  f = {{a->log_probs, a->log_probs_f32}, {a->old_log_probs, a->old_f32}, {a->ref_log_probs, a->ref_f32}, a->advantages,
       a->advantage_per_token, a->ratio_per_sequence, a->mean_per_sequence, a->kl, a->ratio_low, a->ratio_high, a->kl_coef,
       a->entropy_coef};
  q = {a->offsets, a->sequences, a->tokens, a->length, a->mask, a->offsets_i64};
  if (const int rc = seq_check(q)) return rc;
  if ((q.tokens > 0 && !f.lp.p) || (q.count > 0 && q.tokens > 0 && !f.advantages) || f.kl < 0 || f.kl > 3 ||
      (f.whole && f.advantage_tokens))
    return MX_ERR_INVALID_ARG;
  return seq_odd(f.lp) || seq_odd(f.old) || seq_odd(f.ref) || ((uintptr_t)f.advantages & 3) ? MX_ERR_ALIGNMENT : MX_OK;
}

extern "C" int mx_policy_loss(const mx_policy_loss_t* args, float* loss, float* metrics, double* each, void* workspace,
                              void* stream) {
  Policy f;
  Sequences q;
  if (const int rc = policy_check(args, f, q)) return rc;
  if (!loss || !metrics || !workspace) return MX_ERR_INVALID_ARG;
  if (((uintptr_t)loss & 3) || ((uintptr_t)metrics & 3) || ((uintptr_t)each & 7) || ((uintptr_t)workspace & 7)) return MX_ERR_ALIGNMENT;
  seq_loss(f, q, q.count, (double*)workspace, each, loss, metrics, (hipStream_t)stream);
  return status();
}

extern "C" int mx_policy_loss_bwd(const mx_policy_loss_t* args, const double* each, const float* dloss, void* grad, void* stream) {
  Policy f;
  Sequences q;
  if (const int rc = policy_check(args, f, q)) return rc;
  if (q.tokens == 0) return MX_OK;
  if (!each || !dloss || !grad) return MX_ERR_INVALID_ARG;
  if (((uintptr_t)each & 7) || ((uintptr_t)dloss & 3) || ((uintptr_t)grad & (f.lp.f32 ? 3 : 1))) return MX_ERR_ALIGNMENT;
  seq_grads(f, q, each, dloss, grad, (hipStream_t)stream);
  return status();
}

static int preference_check(const mx_preference_loss_t* a, Preference& f, Sequences& q) {
  if (!a) return MX_ERR_INVALID_ARG;
  f = {{a->log_probs, a->log_probs_f32}, {a->ref_log_probs, a->ref_f32}, a->kind, a->mean, a->beta, a->smoothing};
  q = {a->offsets, a->sequences, a->tokens, a->length, a->mask, a->offsets_i64};
  if (const int rc = seq_check(q)) return rc;
  if ((q.tokens > 0 && !f.lp.p) || q.count % 2 || f.kind < 0 || f.kind > 2) return MX_ERR_INVALID_ARG;
  return seq_odd(f.lp) || seq_odd(f.ref) ? MX_ERR_ALIGNMENT : MX_OK;
}

extern "C" int mx_preference_loss(const mx_preference_loss_t* args, float* loss, float* rewards, double* each, void* workspace,
                                  void* stream) {
  Preference f;
  Sequences q;
  if (const int rc = preference_check(args, f, q)) return rc;
  if (!loss || (q.count > 0 && !rewards) || !workspace) return MX_ERR_INVALID_ARG;
  if (((uintptr_t)loss & 3) || ((uintptr_t)rewards & 3) || ((uintptr_t)each & 7) || ((uintptr_t)workspace & 7)) return MX_ERR_ALIGNMENT;
  seq_loss(f, q, q.count / 2, (double*)workspace, each, loss, rewards, (hipStream_t)stream);
  return status();
}

extern "C" int mx_preference_loss_bwd(const mx_preference_loss_t* args, const double* each, const float* dloss, void* grad,
                                      void* stream) {
  Preference f;
  Sequences q;
  if (const int rc = preference_check(args, f, q)) return rc;
  if (q.tokens == 0) return MX_OK;
  if (!each || !dloss || !grad) return MX_ERR_INVALID_ARG;
  if (((uintptr_t)each & 7) || ((uintptr_t)dloss & 3) || ((uintptr_t)grad & (f.lp.f32 ? 3 : 1))) return MX_ERR_ALIGNMENT;
  seq_grads(f, q, each, dloss, grad, (hipStream_t)stream);
  return status();
}
