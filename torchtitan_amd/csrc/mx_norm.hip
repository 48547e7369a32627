// Norms before and after a block, with the block's gate and the residual sum.  For every row of width D, in float32:
//
//   n = h s1 post,  s1 = 1 / sqrt(mean h^2 + eps)       (n = h without a norm behind the block)
//   t = scale r + g n                                    (g n = n without a gate)
//   stream = t,  normed = t s2 pre,  s2 = 1 / sqrt(mean t^2 + eps)
//
// `normed` comes from t before t is rounded to the stream's type.  Backward, from the same h and r, with u = normed's
// gradient times pre:
//
//   e  = dstream + s2 (u - t s2 mean(u t s2)),   dr = scale e,   dpre = sum of rows dnormed t s2
//   dg = sum over the gate's rows of e n,        q = e g
//   dpost = sum of rows q h s1,                  dh = s1 (q post - h s1 mean(q post h s1)); without post dh = q
//
// t is formed again, without the rounding that the stream has.  With post or gate, whose gradients need h, that reads as
// much as the stream would be; for a plain sum it reads one matrix more, and both stay in memory until then.  Without a
// gradient of normed e = dstream and t is not needed.
//
// Sums over rows are float32 parts of one workgroup's rows each, joined in order by a second launch: the same result
// on every run.  Row r of T uses row r / (T / G) of a gate of G rows.
#include <algorithm>

#include "mx_rows.h"

namespace mx {

constexpr int kNormThreads = 256;

// Sum over the workgroup, in every lane; `part` holds a float a wave and may be used again after the next barrier.
template <int THREADS>
__device__ __forceinline__ float group_sum(float v, float* part) {
  v = wave_sum(v);
  if constexpr (THREADS > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) v += part[w];
  }
  return v;
}

// A learned vector, or nothing (then 1 everywhere).
struct NormWeight {
  const void* p;
  int f32;
  __device__ __forceinline__ float at(int64_t i) const {
    return !p ? 1.f : f32 ? ((const float*)p)[i] : bf16_lo(((const uint16_t*)p)[i]);
  }
};

struct NormArgs {
  const void* h;
  const void* r;
  int64_t rows, cols, ldh, ldr;
  NormWeight post, gate, pre;
  int64_t gate_each;  // rows that share a row of the gate
  float scale, eps;
  bool past;          // the matrices written are stored past the caches (see norm_past)
};

template <class T>
__device__ __forceinline__ float norm_element(const T* p) {
  if constexpr (sizeof(T) == 4) return *p;
  else return bf16_lo(*p);
}
template <class T>
__device__ __forceinline__ T norm_rounded(float f) {
  if constexpr (sizeof(T) == 4) return f;
  else return (uint16_t)(__builtin_bit_cast(uint32_t, __builtin_convertvector(v2f_t{f, f}, v2bf_t)));
}

// ---- rows that fit the registers of their lanes: kV-element pieces, piece k of lane l at column (k LANES + l) kV.
// Where the width is no multiple of kV the last piece lies kV in front of the row's end and covers columns of the one
// before again: both lanes form and write the same values there, and the row's sums leave the second out.
constexpr int kV = 8;

template <int LANES, int N>
struct NormShape {
  static constexpr int kLanes = LANES, kPieces = N;              // of one row
  static constexpr int kThreads = LANES > 64 ? LANES : 256;      // of a workgroup
  static constexpr int kRows = kThreads / LANES;                 // that a workgroup works on at a time
  static constexpr int kCols = LANES * N * kV;                   // a row's columns at most
};

// Where a lane's piece lies: from column `at` on, its first `skip` elements another lane's; none if not `in`.
struct NormPlace {
  int at, skip;
  bool in;
};
template <class S>
__device__ __forceinline__ NormPlace norm_place(int k, int lane, int cols) {
  const int c = (k * S::kLanes + lane) * kV;
  const int at = c < cols - kV ? c : cols - kV;
  return {at, c - at, c < cols};
}
template <bool NT, class T>
__device__ __forceinline__ void load_at(const T* row, const NormPlace& p, Piece<T, kV>& q) {
  q = Piece<T, kV>{};
  if (p.in) load_words<NT>(row + p.at, q);
}
template <class T>
__device__ __forceinline__ void store_at(T* row, const NormPlace& p, const float (&f)[kV], bool past = false) {
  if (!p.in) return;
  const Piece<T, kV> q = from_floats<T>(f);
  if (past) store_words<true>(row + p.at, q);
  else store_words<false>(row + p.at, q);
}
__device__ __forceinline__ void weight_at(const NormWeight& w, int64_t row, const NormPlace& p, float (&f)[kV]) {
  if (!w.p) {
#pragma unroll
    for (int e = 0; e < kV; ++e) f[e] = 1.f;
  } else if (w.f32) {
    Piece<float, kV> q;
    load_at<false>((const float*)w.p + row, p, q);
    to_floats(q, f);
  } else {
    Piece<uint16_t, kV> q;
    load_at<false>((const uint16_t*)w.p + row, p, q);
    to_floats(q, f);
  }
}

// The same of a vector that is there, as it lies in memory: nothing waits for it yet.
struct RawWeight {
  uint32_t w[kV];
};
__device__ __forceinline__ RawWeight raw_weight(const NormWeight& w, int64_t row, const NormPlace& p) {
  RawWeight raw{};
  if (w.f32) {
    Piece<float, kV> q;
    load_at<false>((const float*)w.p + row, p, q);
#pragma unroll
    for (int i = 0; i < kV; ++i) raw.w[i] = q.w[i];
  } else {
    Piece<uint16_t, kV> q;
    load_at<false>((const uint16_t*)w.p + row, p, q);
#pragma unroll
    for (int i = 0; i < kV / 2; ++i) raw.w[i] = q.w[i];
  }
  return raw;
}
__device__ __forceinline__ void raw_floats(const NormWeight& w, const RawWeight& raw, float (&f)[kV]) {
#pragma unroll
  for (int e = 0; e < kV; ++e) f[e] = __uint_as_float(w.f32 ? raw.w[e] : e & 1 ? raw.w[e / 2] & 0xFFFF0000u : raw.w[e / 2] << 16);
}

// gate * post: what a row's normalised block output is multiplied with.
__device__ __forceinline__ void side_at(const NormArgs& a, int64_t g0, const NormPlace& p, float (&f)[kV]) {
  float q[kV];
  weight_at(a.post, 0, p, q);
  weight_at(a.gate, g0, p, f);
#pragma unroll
  for (int e = 0; e < kV; ++e) f[e] *= q[e];
}

// Sum over the lanes of a row, in each of them.  Rows of more than a wave go through `part`, a float a wave, with one
// barrier: whoever comes by here again before another barrier brings another `part`.
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v, float* part) {
  v += __uint_as_float(dpp<kQuadXor1>(__float_as_uint(v)));
  v += __uint_as_float(dpp<kQuadXor2>(__float_as_uint(v)));
  v += __uint_as_float(dpp<kRowHalfMirror>(__float_as_uint(v)));
  v += __uint_as_float(dpp<kRowMirror>(__float_as_uint(v)));  // (16 lanes)
  if constexpr (LANES == 32) v += __shfl_xor(v, 16, 64);
  if constexpr (LANES >= 64) {
    auto of = [&](int lane) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), lane)); };
    v = (of(0) + of(16)) + (of(32) + of(48));
  }
  if constexpr (LANES > 64) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < LANES / 64; ++w) v += part[w];
  }
  return v;
}

// 1 / sqrt(x), x >= 0: the hardware's, which takes no denormals, and a Newton step on its remainder, which brings it to
// within an ulp (none for 0 and infinity, whose remainder is NaN).
__device__ __forceinline__ float norm_rsqrt(float x) {
  const bool tiny = x < 0x1p-100f;
  const float y = tiny ? x * 0x1p100f : x, s = __builtin_amdgcn_rsqf(y), rest = __builtin_fmaf(-y * s, s, 1.f);
  const float best = rest == rest ? __builtin_fmaf(0.5f * s, rest, s) : s;
  return tiny ? best * 0x1p50f : best;
}

// Sum of a * b over a lane's pieces of a row; `ragged`: the width is no multiple of kV, and elements may be another
// lane's.
template <int N>
__device__ __forceinline__ float own_products(const float (&a)[N][kV], const float (&b)[N][kV], const NormPlace (&at)[N],
                                              bool ragged) {
  float sum = 0.f;
  if (ragged) {
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
      for (int e = 0; e < kV; ++e)  // (the product is left out, not made zero: infinity times 0 is no zero)
        sum = e >= at[k].skip ? __builtin_fmaf(a[k][e], b[k][e], sum) : sum;
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
      for (int e = 0; e < kV; ++e) sum = __builtin_fmaf(a[k][e], b[k][e], sum);
  }
  return sum;
}

// A workgroup takes every gridDim.x-th row, or `pair` rows that lie together (kRows times as many); the next row is on its
// way while one is worked on, and the weights stay in registers (with two pieces a lane they are read for every row).
// Bound by memory: 16384 x 4096 with both norms and a gate 97 us (5.5 TB/s; 83 where the last cache has h and r already),
// 147456 x 2048 419 to 440 (5.5 to 5.8, of the 6.2 that two matrices read and two written reach without any arithmetic).
template <class S, class H, class R>
__global__ __launch_bounds__(S::kThreads) void residual_norm_kernel(NormArgs a, int pair, R* __restrict__ stream,
                                                                    H* __restrict__ normed, float* __restrict__ rstd) {
  constexpr int N = S::kPieces;
  constexpr bool kHeld = N == 1;
  __shared__ float part[2][2][S::kLanes / 64 + 1];  // (two rows' worth: see lanes_sum)
  const int lane = threadIdx.x % S::kLanes;
  const int64_t step = pair ? S::kRows : (int64_t)gridDim.x * S::kRows, begin = (int64_t)blockIdx.x * S::kRows * (pair ? pair : 1);
  int64_t row = begin + threadIdx.x / S::kLanes;
  const int64_t end = pair && begin + S::kRows * pair < a.rows ? begin + S::kRows * pair : a.rows;
  if (row >= end) return;  // (whole workgroups where rows share barriers)
  struct Row {
    Piece<H, kV> h[N];
    Piece<R, kV> r[N];
  };
  NormPlace at[N];
#pragma unroll
  for (int k = 0; k < N; ++k) at[k] = norm_place<S>(k, lane, (int)a.cols);
  auto fetch = [&](Row& q, int64_t i) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      load_at<true>((const H*)a.h + i * a.ldh, at[k], q.h[k]);
      load_at<true>((const R*)a.r + i * a.ldr, at[k], q.r[k]);
    }
  };
  Row now, next;
  fetch(now, row);
  // pre, and gate * post, of piece k
  const bool ragged = a.cols % kV != 0;
  const float per = 1.f / (float)a.cols;
  float side1[kV], pre1[kV];
  int64_t group = -1;
  if constexpr (kHeld) weight_at(a.pre, 0, at[0], pre1);
  for (int turn = 0;; turn ^= 1) {
    const int64_t coming = row + step;
    if (coming < end) fetch(next, coming);
    const int64_t g = a.gate.p ? (uint32_t)row / (uint32_t)a.gate_each : 0;  // (rows fit 31 bits)
    if (kHeld && g != group) side_at(a, g * a.cols, at[0], side1);
    group = g;
    float x[N][kV], s1 = 1.f, s2 = 1.f;
#pragma unroll
    for (int k = 0; k < N; ++k) to_floats(now.h[k], x[k]);
    if (a.post.p) s1 = norm_rsqrt(__builtin_fmaf(lanes_sum<S::kLanes>(own_products(x, x, at, ragged), part[turn][0]), per, a.eps));
#pragma unroll
    for (int k = 0; k < N; ++k) {
      float y[kV], w[kV];
      to_floats(now.r[k], y);
      if constexpr (!kHeld) side_at(a, g * a.cols, at[k], w);
#pragma unroll
      for (int e = 0; e < kV; ++e) x[k][e] = __builtin_fmaf(a.scale, y[e], x[k][e] * s1 * (kHeld ? side1[e] : w[e]));
      store_at(stream + row * a.cols, at[k], x[k], a.past);
    }
    if (a.pre.p) {
      s2 = norm_rsqrt(__builtin_fmaf(lanes_sum<S::kLanes>(own_products(x, x, at, ragged), part[turn][1]), per, a.eps));
#pragma unroll
      for (int k = 0; k < N; ++k) {
        float w[kV];
        if constexpr (!kHeld) weight_at(a.pre, 0, at[k], w);
#pragma unroll
        for (int e = 0; e < kV; ++e) x[k][e] = x[k][e] * s2 * (kHeld ? pre1[e] : w[e]);
        store_at(normed + row * a.cols, at[k], x[k], a.past);
      }
    }
    if (rstd && lane == 0) {
      rstd[row] = s1;
      rstd[a.rows + row] = s2;
    }
    if (coming >= end) break;
    row = coming;
    now = next;
  }
}

// Rows of any width (below 8 and above 16384 columns), one workgroup a row, element by element; what a later step needs of an
// earlier one is formed again: 2048 x 20000 231 us forward and 1355 backward, limited by the instructions of the repeated work.
template <int THREADS, class H, class R>
__global__ __launch_bounds__(THREADS) void residual_norm_any_kernel(NormArgs a, R* __restrict__ stream,
                                                                         H* __restrict__ normed, float* __restrict__ rstd) {
  __shared__ float part[THREADS / 64];
  const int64_t row = blockIdx.x;
  const H* h = (const H*)a.h + row * a.ldh;
  const R* r = (const R*)a.r + row * a.ldr;
  const int64_t g0 = row / a.gate_each * a.cols;
  float s1 = 1.f, s2 = 1.f, sum = 0.f;
  if (a.post.p) {
    for (int64_t c = threadIdx.x; c < a.cols; c += THREADS) {
      const float x = norm_element(h + c);
      sum += x * x;
    }
    s1 = 1.f / sqrtf(group_sum<THREADS>(sum, part) / (float)a.cols + a.eps);
  }
  auto total = [&](int64_t c) {
    return a.scale * norm_element(r + c) + a.gate.at(g0 + c) * (norm_element(h + c) * s1 * a.post.at(c));
  };
  sum = 0.f;
  for (int64_t c = threadIdx.x; c < a.cols; c += THREADS) {
    const float t = total(c);
    stream[row * a.cols + c] = norm_rounded<R>(t);
    sum += t * t;
  }
  if (a.pre.p) {
    s2 = 1.f / sqrtf(group_sum<THREADS>(sum, part) / (float)a.cols + a.eps);
    for (int64_t c = threadIdx.x; c < a.cols; c += THREADS)
      normed[row * a.cols + c] = norm_rounded<H>(total(c) * s2 * a.pre.at(c));
  }
  if (rstd && threadIdx.x == 0) {
    rstd[row] = s1;
    rstd[a.rows + row] = s2;
  }
}

// How the rows are dealt out in the backward pass: `strips` workgroups' worth to every row of the gate, which take its
// rows in turn, so that the chip works its way through memory in order (16384 x 4096: 133 us, with strips of rows that
// lie together 150); a workgroup takes every gridDim.x-th strip.
// `run`: workgroup b, which runs on XCD b mod 8, takes the strips as if `run` of them were dealt to one XCD after the
// other; 1: in the order of b.
struct NormStrips {
  int64_t strips, total;
  unsigned run;
  __device__ __forceinline__ int64_t mine() const {
    const unsigned b = blockIdx.x;
    return (int64_t)(b / (8 * run)) * (8 * run) + b % 8 * run + b / 8 % run;
  }
};

struct NormGrads {
  const void* dstream;
  const void* dnormed;
  void* dh;
  void* dr;
  float* rows_part;  // [workgroups][3][cols]: sums of post, pre and, one strip at a time, of the gate
  float* gate_part;  // [strips in all][cols], where a row of the gate has more than one
  void* dgate;
  int dgate_f32;
};

template <int THREADS, class H, class R>
__global__ __launch_bounds__(THREADS) void residual_norm_bwd_any_kernel(NormArgs a, NormStrips strips,
                                                                             const float* __restrict__ rstd, NormGrads o) {
  __shared__ float part[THREADS / 64];
  float* dpost = o.rows_part + (int64_t)blockIdx.x * 3 * a.cols;
  float* dpre = dpost + a.cols;
  float* dgate = o.dgate ? dpre + a.cols : nullptr;
  for (int64_t c = threadIdx.x; c < a.cols; c += THREADS) dpost[c] = dpre[c] = 0.f;
  const float width = (float)a.cols;
  for (int64_t strip = blockIdx.x; strip < strips.total; strip += gridDim.x) {
    const int64_t group = strip / strips.strips, first = group * a.gate_each + strip - group * strips.strips;
    const int64_t g0 = group * a.cols;
    if (dgate)
      for (int64_t c = threadIdx.x; c < a.cols; c += THREADS) dgate[c] = 0.f;
    for (int64_t row = first; row < (group + 1) * a.gate_each; row += strips.strips) {
      const H* h = (const H*)a.h + row * a.ldh;
      const R* r = (const R*)a.r + row * a.ldr;
      const R* ds = o.dstream ? (const R*)o.dstream + row * a.cols : nullptr;
      const H* dy = o.dnormed ? (const H*)o.dnormed + row * a.cols : nullptr;
      const float s1 = rstd[row], s2 = rstd[a.rows + row];
      auto branch = [&](int64_t c) { return norm_element(h + c) * s1 * a.post.at(c); };
      auto hat = [&](int64_t c) { return (a.scale * norm_element(r + c) + a.gate.at(g0 + c) * branch(c)) * s2; };
      float mean = 0.f;
      if (dy) {
        for (int64_t c = threadIdx.x; c < a.cols; c += THREADS) mean += norm_element(dy + c) * a.pre.at(c) * hat(c);
        mean = group_sum<THREADS>(mean, part) / width;
      }
      auto inner = [&](int64_t c) {
        const float e = ds ? norm_element(ds + c) : 0.f;
        return dy ? e + s2 * (norm_element(dy + c) * a.pre.at(c) - hat(c) * mean) : e;
      };
      float sum = 0.f;
      for (int64_t c = threadIdx.x; c < a.cols; c += THREADS) {
        const float e = inner(c), q = e * a.gate.at(g0 + c), hs = norm_element(h + c) * s1;
        if (o.dr) ((R*)o.dr)[row * a.cols + c] = norm_rounded<R>(a.scale * e);
        if (dy) dpre[c] += norm_element(dy + c) * hat(c);
        if (dgate) dgate[c] += e * branch(c);
        if (a.post.p) dpost[c] += q * hs;
        sum += q * a.post.at(c) * hs;
      }
      if (o.dh) {
        if (a.post.p) sum = group_sum<THREADS>(sum, part) / width;
        for (int64_t c = threadIdx.x; c < a.cols; c += THREADS) {
          const float q = inner(c) * a.gate.at(g0 + c);
          const float d = a.post.p ? s1 * (q * a.post.at(c) - norm_element(h + c) * s1 * sum) : q;
          ((H*)o.dh)[row * a.cols + c] = norm_rounded<H>(d);
        }
      }
    }
    if (dgate)
      for (int64_t c = threadIdx.x; c < a.cols; c += THREADS) {
        if (strips.strips > 1) o.gate_part[strip * a.cols + c] = dgate[c];
        else if (o.dgate_f32) ((float*)o.dgate)[group * a.cols + c] = dgate[c];
        else ((uint16_t*)o.dgate)[group * a.cols + c] = norm_rounded<uint16_t>(dgate[c]);
      }
  }
}

// A lane's sums of all rows of its workgroup: the rows' lanes add theirs to `lds` in turn.
template <class S>
__device__ __forceinline__ void rows_joined(float (&acc)[S::kPieces][kV], float* lds) {
  if constexpr (S::kRows > 1) {
    const int lane = threadIdx.x % S::kLanes, sub = threadIdx.x / S::kLanes;
    for (int s = 0; s < S::kRows; ++s) {
      if (sub == s) {
#pragma unroll
        for (int k = 0; k < S::kPieces; ++k)
#pragma unroll
          for (int e = 0; e < kV; ++e) {
            float* at = lds + (k * kV + e) * S::kLanes + lane;  // (lanes side by side: no bank conflicts)
            if (s > 0) acc[k][e] += *at;
            *at = acc[k][e];
          }
      }
      __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < S::kPieces; ++k)
#pragma unroll
      for (int e = 0; e < kV; ++e) acc[k][e] = lds[(k * kV + e) * S::kLanes + lane];
    __syncthreads();
  }
}

// SIDE: the block's side of the sum (norm behind it, gate) as well; else h has the gradient e.  Over the rows of a strip,
// which share a row of the gate, both weights of that side need the same sum of e h s1: times post it is the gate's
// gradient, times the gate post's.
// SOLO: the lanes of a row take strips of their own (see norm_solo), of a row of the gate each; the next strip's first row
// and gate are on their way while one is worked on.
// NORMED: normed has a gradient.  Without one e is dstream as it is: nothing of t, which may be infinite, is in the
// result, and neither residual nor a sum over the row is needed for it.  us with one / without, 16384 x 4096: norm and gate
// 139 / 90 (5.8 and 6.0 TB/s), the norm alone 89, the plain sum 63; 147456 x 2048 708 / 546; 8192 x 16384 428 / 225.
template <class S, bool SIDE, bool SOLO, bool NORMED, class H, class R>
__global__ __launch_bounds__(S::kThreads) void residual_norm_bwd_kernel(NormArgs a, NormStrips strips,
                                                                        const float* __restrict__ rstd, NormGrads o) {
  constexpr int N = S::kPieces;
  constexpr bool kHeld = N == 1;  // (as above)
  __shared__ float part[2][2][S::kLanes / 64 + 1];
  __shared__ float lds[S::kRows > 1 ? S::kCols : 1];
  const int lane = threadIdx.x % S::kLanes, sub = threadIdx.x / S::kLanes;
  const float per = 1.f / (float)a.cols;
  struct Row {
    Piece<H, kV> h[N], dy[N];
    Piece<R, kV> r[N], ds[N];
    float s1 = 1.f, s2 = 1.f;
  };
  NormPlace at[N];
#pragma unroll
  for (int k = 0; k < N; ++k) at[k] = norm_place<S>(k, lane, (int)a.cols);
  auto fetch = [&](Row& q, int64_t i) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      if constexpr (SIDE || NORMED) load_at<true>((const H*)a.h + i * a.ldh, at[k], q.h[k]);
      if constexpr (NORMED) {
        load_at<true>((const R*)a.r + i * a.ldr, at[k], q.r[k]);
        load_at<true>((const H*)o.dnormed + i * a.cols, at[k], q.dy[k]);
      }
      q.ds[k] = Piece<R, kV>{};
      if (o.dstream) load_at<true>((const R*)o.dstream + i * a.cols, at[k], q.ds[k]);
    }
    if constexpr (SIDE || NORMED) q.s1 = rstd[i];
    if constexpr (NORMED) q.s2 = rstd[a.rows + i];
  };
  // pre, and gate * post of the strip, of piece k
  float pre1[kV], side1[kV];
  auto pre_at = [&](int k, float (&f)[kV]) { weight_at(a.pre, 0, at[k], f); };
  const bool ragged = a.cols % kV != 0;
  if constexpr (kHeld && NORMED) pre_at(0, pre1);
  float dpre[N][kV] = {}, dpost[N][kV] = {};
  int turn = 0;
  constexpr int kTogether = SOLO ? 1 : S::kRows;  // rows that a strip takes at a time
  constexpr int kStrips = S::kRows / kTogether;   // strips that a workgroup takes at a time
  const int mine = SOLO ? 0 : sub;
  Row now, next;
  bool fetched = false;  // `now` and the gate, by the strip before
  RawWeight gate_next;
  float gate1[kV], post1[kV];
  if constexpr (SOLO) weight_at(a.post, 0, at[0], post1);
  for (int64_t strip = strips.mine() * kStrips + (SOLO ? sub : 0); strip < strips.total; strip += (int64_t)gridDim.x * kStrips) {
    const int64_t group = (uint32_t)strip / (uint32_t)strips.strips, first = group * a.gate_each + (strip - group * strips.strips) * kTogether;
    const int64_t end = (group + 1) * a.gate_each, hop = strips.strips * kTogether;
    const int64_t g0 = group * a.cols;
    float both[N][kV] = {};
    int64_t row = first + mine;
    if (kHeld && !fetched && row < end) fetch(now, row);
    if constexpr (SOLO) {
      raw_floats(a.gate, fetched ? gate_next : raw_weight(a.gate, g0, at[0]), gate1);
#pragma unroll
      for (int e = 0; e < kV; ++e) side1[e] = gate1[e] * post1[e];
    } else if constexpr (kHeld && SIDE) {
      side_at(a, g0, at[0], side1);
    }
    fetched = false;
    for (; row < end; row += hop, turn ^= 1) {
      if constexpr (!kHeld) fetch(now, row);
      if constexpr (kHeld) {
        if (row + hop < end) fetch(next, row + hop);
        else if (SOLO && strip + gridDim.x * kStrips < strips.total) {
          const int64_t strip2 = strip + gridDim.x * kStrips, group2 = (uint32_t)strip2 / (uint32_t)strips.strips;
          const int64_t row2 = group2 * a.gate_each + (strip2 - group2 * strips.strips) * kTogether + mine;
          if (row2 < (group2 + 1) * a.gate_each) {
            fetch(next, row2);
            gate_next = raw_weight(a.gate, group2 * a.cols, at[0]);
            fetched = true;
          }
        }
      }
      const float s1 = now.s1, s2 = now.s2;
      if constexpr (!kHeld)  // (nothing of the weights is kept from row to row: 8192 x 16384 412 us, where what was kept spilled 975)
#pragma unroll
        for (int k = 0; k < N; ++k) asm volatile("" : "+v"(at[k].at));
      float hat[N][kV], u[N][kV], mean = 0.f;
      if constexpr (NORMED) {
#pragma unroll
        for (int k = 0; k < N; ++k) {
          float x[kV], y[kV], d[kV], w[kV];
          to_floats(now.h[k], x);
          to_floats(now.r[k], y);
          to_floats(now.dy[k], d);
          if constexpr (SIDE) {
            if constexpr (!kHeld) side_at(a, g0, at[k], w);
#pragma unroll
            for (int e = 0; e < kV; ++e) x[e] = x[e] * s1 * (kHeld ? side1[e] : w[e]);
          }
          if constexpr (!kHeld) pre_at(k, w);
#pragma unroll
          for (int e = 0; e < kV; ++e) {
            hat[k][e] = __builtin_fmaf(a.scale, y[e], x[e]) * s2;
            dpre[k][e] = __builtin_fmaf(d[e], hat[k][e], dpre[k][e]);
            u[k][e] = d[e] * (kHeld ? pre1[e] : w[e]);
          }
        }
        mean = lanes_sum<S::kLanes>(own_products(u, hat, at, ragged), part[turn][0]) * per;
      }
      float (&q)[N][kV] = u;  // (in place: what h's gradient is formed from)
#pragma unroll
      for (int k = 0; k < N; ++k) {
        float w[kV], e1[kV], dr[kV];
        to_floats(now.ds[k], e1);
#pragma unroll
        for (int e = 0; e < kV; ++e) {
          if constexpr (NORMED) e1[e] = __builtin_fmaf(s2, __builtin_fmaf(-hat[k][e], mean, u[k][e]), e1[e]);
          dr[e] = a.scale * e1[e];
        }
        if (o.dr) store_at((R*)o.dr + row * a.cols, at[k], dr, a.past);
        if constexpr (SIDE) {
          float x[kV];
          to_floats(now.h[k], x);
          if constexpr (!kHeld) side_at(a, g0, at[k], w);
#pragma unroll
          for (int e = 0; e < kV; ++e) {
            hat[k][e] = x[e] * s1;  // (h's share from here on)
            both[k][e] = __builtin_fmaf(e1[e], hat[k][e], both[k][e]);
            q[k][e] = e1[e] * (kHeld ? side1[e] : w[e]);
          }
        } else {
          if (o.dh) store_at((H*)o.dh + row * a.cols, at[k], e1, a.past);
        }
      }
      if constexpr (SIDE) {
        if (a.post.p) {  // (else q is the gradient: h, which may be infinite, is not in it)
          const float mean1 = lanes_sum<S::kLanes>(own_products(q, hat, at, ragged), part[turn][1]) * per;
#pragma unroll
          for (int k = 0; k < N; ++k)
#pragma unroll
            for (int e = 0; e < kV; ++e) q[k][e] = s1 * __builtin_fmaf(-hat[k][e], mean1, q[k][e]);
        }
        if (o.dh) {
#pragma unroll
          for (int k = 0; k < N; ++k) store_at((H*)o.dh + row * a.cols, at[k], q[k], a.past);
        }
      }
      if constexpr (kHeld) now = next;
    }
    if constexpr (SIDE) {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        float g[kV];
        if constexpr (!SOLO) weight_at(a.gate, g0, at[k], g);
#pragma unroll
        for (int e = 0; e < kV; ++e) dpost[k][e] = __builtin_fmaf(SOLO ? gate1[e] : g[e], both[k][e], dpost[k][e]);
      }
      if (o.dgate) {
        if constexpr (!SOLO) rows_joined<S>(both, lds);
        if (SOLO || sub == 0) {
#pragma unroll
          for (int k = 0; k < N; ++k) {
            float p[kV];
            if constexpr (!SOLO) weight_at(a.post, 0, at[k], p);
#pragma unroll
            for (int e = 0; e < kV; ++e) p[e] = (SOLO ? post1[e] : p[e]) * both[k][e];
            if (strips.strips > 1) store_at(o.gate_part + strip * a.cols, at[k], p);
            else if (o.dgate_f32) store_at((float*)o.dgate + g0, at[k], p);
            else store_at((uint16_t*)o.dgate + g0, at[k], p);
          }
        }
      }
    }
  }
  float* out = o.rows_part + (int64_t)blockIdx.x * 3 * a.cols;
  rows_joined<S>(dpre, lds);
  if constexpr (SIDE) rows_joined<S>(dpost, lds);
  if (sub == 0) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      store_at(out + a.cols, at[k], dpre[k]);
      if constexpr (SIDE) store_at(out, at[k], dpost[k]);
    }
  }
}

// Sums of the workgroups' parts: blockIdx.y 0 post, 1 pre, from 2 on the rows of the gate, those without a place left
// out.  A workgroup takes 64 columns; 16 lanes of four columns each, 16 such groups that take every 16th part, in order.
struct NormJoin {
  const float* rows_part;
  const float* gate_part;
  int64_t groups, strips;
  void* out[3];
  int f32[3];
};
__global__ __launch_bounds__(kNormThreads) void residual_norm_join_kernel(NormJoin j, int64_t cols) {
  constexpr int kEach = 16;
  __shared__ float sums[kEach][64];
  const int which = blockIdx.y < 2 ? (int)blockIdx.y : 2;
  if (!j.out[which]) return;
  const int64_t g = which == 2 ? (int64_t)blockIdx.y - 2 : 0;
  const int lane = threadIdx.x & 15, slice = threadIdx.x >> 4;
  const int64_t c = (int64_t)blockIdx.x * 64 + lane * 4, left = cols - c;
  const float* part = which == 2 ? j.gate_part + g * j.strips * cols : j.rows_part + which * cols;
  const int64_t parts = which == 2 ? j.strips : j.groups, stride = which == 2 ? cols : 3 * cols;
  float acc[4] = {};
#pragma unroll 8
  for (int64_t p = slice; p < parts; p += kEach) {
    Piece<float, 4> q;
    load_piece<false>(part + p * stride + c, left, q);
    float f[4];
    to_floats(q, f);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] += f[e];
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) sums[slice][lane * 4 + e] = acc[e];
  __syncthreads();
  const int64_t col = (int64_t)blockIdx.x * 64 + threadIdx.x;
  if (threadIdx.x < 64 && col < cols) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < kEach; ++k) s += sums[k][threadIdx.x];
    if (j.f32[which]) ((float*)j.out[which])[g * cols + col] = s;
    else ((uint16_t*)j.out[which])[g * cols + col] = norm_rounded<uint16_t>(s);
  }
}

// Stores go past the caches where two matrices of this size do not stay in the last one (256 MB) until the next operator
// reads them.  us forward and backward, past / through: 16384 x 4096 (2 x 134 MB) 89 + 162 / 85 + 144; x 8192 196 + 323 /
// 212 + 339; 147456 x 2048 424 + 663 / 445 + 704.
static bool norm_past(int64_t elements, int h_f32, int r_f32) { return elements * (2 * (2 + !!h_f32 + !!r_f32)) > (384 << 20); }

// Calls f(shape) with the smallest shape that holds a row (640 and 768 lanes: 16384 x 5120 265 -> 192 us backward, x 6144 274 ->
// 229, some of it by a workgroup for every CU; 896 lanes gain nothing over 1024), or f(threads) for rows that none does.
template <class S>
constexpr bool norm_shaped = false;
template <int LANES, int N>
constexpr bool norm_shaped<NormShape<LANES, N>> = true;
template <class F>
static void norm_shape(int64_t cols, F&& f) {
  if (cols < kV) f(std::integral_constant<int, 64>());
  else if (cols <= NormShape<16, 1>::kCols) f(NormShape<16, 1>());
  else if (cols <= NormShape<32, 1>::kCols) f(NormShape<32, 1>());
  else if (cols <= NormShape<64, 1>::kCols) f(NormShape<64, 1>());
  else if (cols <= NormShape<128, 1>::kCols) f(NormShape<128, 1>());
  else if (cols <= NormShape<256, 1>::kCols) f(NormShape<256, 1>());
  else if (cols <= NormShape<512, 1>::kCols) f(NormShape<512, 1>());
  else if (cols <= NormShape<640, 1>::kCols) f(NormShape<640, 1>());
  else if (cols <= NormShape<768, 1>::kCols) f(NormShape<768, 1>());
  else if (cols <= NormShape<1024, 1>::kCols) f(NormShape<1024, 1>());
  else if (cols <= NormShape<1024, 2>::kCols) f(NormShape<1024, 2>());
  else f(std::integral_constant<int, 1024>());
}

// Workgroups of `waves` waves for every CU, one at least (16384 x 8192 with the block's side 297 us, with one for two CUs 322; 8192 x
// 16384 412 and 603).
static int64_t norm_groups(int64_t cols, int waves) {
  int threads = 0;
  norm_shape(cols, [&](auto shape) {
    using S = decltype(shape);
    if constexpr (norm_shaped<S>) threads = S::kThreads;
    else threads = S::value;
  });
  return 256 * std::max(1, 64 * waves / threads);
}
// Forward: as many workgroups as stay resident come back for more rows; matrices that the last cache does not hold are
// gone through in order, two rows a workgroup, up to 2048 columns.  us in turn / two rows: 147456 x 2048 461 / 419, 65536 x
// 1024 (past no cache) 83 / 92, 73728 x 4096 448 / 460, 16384 x 8192 218 / 238.  16 waves a CU stay, of workgroups of more than
// 512 lanes two: 16384 x 5120 136 us with one, 123 with two, 141 with three; x 6144 164 and 149; x 4096 83, with twice as
// many 93.
// A launch has fewer than 2^32 lanes: more rows than two a workgroup reach by that (2^29 of 128 columns) are taken in turn.
constexpr int kNormPair = 2;
template <class S>
static int64_t norm_pairs(const NormArgs& a) { return (a.rows + S::kRows * kNormPair - 1) / (S::kRows * kNormPair); }
template <class S>
static int norm_pair(const NormArgs& a) {
  return a.past && a.cols <= 2048 && norm_pairs<S>(a) * S::kThreads < (int64_t{1} << 32) ? kNormPair : 0;
}
template <class S>
static int64_t norm_fwd_groups(const NormArgs& a) {
  if (norm_pair<S>(a)) return norm_pairs<S>(a);
  return std::min<int64_t>((a.rows + S::kRows - 1) / S::kRows, norm_groups(a.cols, S::kThreads > 512 ? S::kThreads / 32 : 16));
}

// The backward pass, waves a CU: with the block's side the 8 that its registers allow, without it 16, or 8 for narrow rows.  With
// the block's side and matrices that the last cache does not hold as many workgroups as bring 6 waves' worth of columns, one at least: the
// fewer are on their way, the better they stay in the order of memory (147456 x 2048 768 -> 649 us, x 1024 358 -> 332, 300000 x 512
// 367 -> 327; 32768 x 2048, which it nearly holds, 138 -> 150).
static int64_t norm_bwd_groups(int64_t cols, bool side, bool past) {
  if (!side) return norm_groups(cols, cols <= 2048 ? 8 : 16);
  const int64_t most = norm_groups(cols, 8);
  if (!past) return most;
  int64_t together = 1;
  norm_shape(cols, [&](auto shape) {
    if constexpr (norm_shaped<decltype(shape)>) together = decltype(shape)::kRows;
  });
  return std::min(most, 256 * std::max<int64_t>(1, 6 * 64 * kV / (cols * together)));
}

// Strips for each row's lanes, for rows of the gate that have few rows themselves.  Where a workgroup takes several rows at
// a time: if they work through their rows sooner so than together.  Where it takes one: up to 4 rows of one gate.  us
// shared / so: 65536 x 512 with a gate for every row 394 / 108, x 1024 309 / 227, 16384 x 4096 277 / 216 and for every 4 rows
// 170 / 169.  Rows of more lanes have no registers for it (8192 x 8192 392 / 466).
template <class S>
constexpr bool norm_solo_shape() {
  return S::kPieces == 1 && S::kLanes <= 512;
}
static bool norm_solo(int64_t rows, int64_t gate_rows, int64_t groups, int64_t together) {
  auto up = [](int64_t x, int64_t y) { return (x + y - 1) / y; };
  const int64_t each = rows / gate_rows;
  if (together == 1) return each <= 4;
  return up(gate_rows, groups * together) * each < up(gate_rows, groups) * up(each, together);
}

struct NormBwdPlan {
  NormStrips strips;
  int64_t groups;
  bool solo;
};
static NormBwdPlan norm_bwd_plan(int64_t rows, int64_t cols, int64_t gate_rows, bool side, bool gate, bool past) {
  int64_t together = 0;
  norm_shape(cols, [&](auto shape) {
    if constexpr (norm_shaped<decltype(shape)>) {
      if (norm_solo_shape<decltype(shape)>()) together = decltype(shape)::kRows;
    }
  });
  // (with more gates than CUs the rows are in no such order: 147456 x 2048 with a gate each 1422 -> 929 us)
  const int64_t groups = norm_bwd_groups(cols, side, past && gate_rows <= 256), strips = std::max<int64_t>(1, std::min(groups, rows) / gate_rows);
  const bool solo = gate && strips == 1 && together > 0 && norm_solo(rows, gate_rows, groups, together);
  const int64_t total = strips * gate_rows, units = solo ? (total + together - 1) / together : total;
  // Matrices that the last cache does not hold: an XCD's strips lie together, an eighth of them all, with the block's side and one
  // gate eight.  us in the order of b / by eighths / by eights: 147456 x 2048 with 16 gates 707 / 696 / 726, without the block's side 690 /
  // 687 / 707, 73728 x 4096 without it 716 / 673 / 704, with it 804 / 796 / 717, 16384 x 8192 298 / 296 / 288.
  const int64_t used = std::min(units, groups), run = !past ? 1 : side && gate_rows == 1 ? 8 : used / 8;
  return {{strips, total, (unsigned)(run > 0 && used % (8 * run) == 0 ? run : 1)}, used, solo};
}

template <class F>
static void norm_types(int h_f32, int r_f32, F&& f) {
  if (h_f32) f(float(), float());
  else if (r_f32) f(uint16_t(), float());
  else f(uint16_t(), uint16_t());
}

static int norm_check(const void* h, int h_f32, const void* r, int r_f32, int64_t rows, int64_t cols, int64_t ldh,
                      int64_t ldr, const void* post, const void* gate, const void* pre, int weights_f32, int64_t gate_rows) {
  if (rows < 0 || cols < 0 || (rows > 1 && (ldh < cols || ldr < cols)) || (h_f32 && !r_f32)) return MX_ERR_INVALID_ARG;
  if (gate_rows < 1 || (rows > 0 && rows % gate_rows)) return MX_ERR_INVALID_ARG;
  if (rows == 0 || cols == 0) return MX_OK;
  if (!h || !r) return MX_ERR_INVALID_ARG;
  auto odd = [](const void* p, int f32) { return ((uintptr_t)p & (f32 ? 3 : 1)) != 0; };
  if (odd(h, h_f32) || odd(r, r_f32) || odd(post, weights_f32 & 1) || odd(gate, weights_f32 & 2) || odd(pre, weights_f32 & 4))
    return MX_ERR_ALIGNMENT;
  // (a launch has fewer than 2^32 lanes: rows with a workgroup each)
  const bool any = cols < kV || cols > NormShape<1024, 2>::kCols;
  if (rows > (any ? 0x3FFFFF : 0x7FFFFFFF) || cols > 0x7FFFFFFF) return MX_ERR_UNSUPPORTED;
  return MX_OK;
}

}  // namespace mx

using namespace mx;

extern "C" int mx_residual_norm(const void* h, int h_f32, const void* r, int r_f32, int64_t rows, int64_t cols, int64_t ldh,
                                int64_t ldr, const void* post, const void* gate, const void* pre, int weights_f32,
                                int64_t gate_rows, float scale, float eps, void* stream_out, void* normed, float* rstd,
                                void* stream) {
  if (const int rc = norm_check(h, h_f32, r, r_f32, rows, cols, ldh, ldr, post, gate, pre, weights_f32, gate_rows)) return rc;
  if (rows == 0 || cols == 0) return MX_OK;
  if (!stream_out || (pre && !normed)) return MX_ERR_INVALID_ARG;
  if (((uintptr_t)stream_out & (r_f32 ? 3 : 1)) || ((uintptr_t)normed & (h_f32 ? 3 : 1)) || ((uintptr_t)rstd & 3))
    return MX_ERR_ALIGNMENT;
  const NormArgs a{h, r, rows, cols, ldh, ldr, {post, weights_f32 & 1}, {gate, weights_f32 & 2}, {pre, weights_f32 & 4},
                   rows / gate_rows, scale, eps, norm_past(rows * cols, h_f32, r_f32)};
  norm_types(h_f32, r_f32, [&](auto ht, auto rt) {
    using H = decltype(ht);
    using R = decltype(rt);
    norm_shape(cols, [&](auto shape) {
      using S = decltype(shape);
      if constexpr (!norm_shaped<S>)
        hipLaunchKernelGGL((residual_norm_any_kernel<S::value, H, R>), dim3((unsigned)rows), dim3(S::value), 0,
                           (hipStream_t)stream, a, (R*)stream_out, (H*)normed, rstd);
      else
        hipLaunchKernelGGL((residual_norm_kernel<S, H, R>), dim3((unsigned)norm_fwd_groups<S>(a)), dim3(S::kThreads), 0,
                           (hipStream_t)stream, a, norm_pair<S>(a), (R*)stream_out, (H*)normed, rstd);
    });
  });
  return hipGetLastError() == hipSuccess ? MX_OK : MX_ERR_LAUNCH;
}

extern "C" int64_t mx_residual_norm_workspace(int64_t rows, int64_t cols, int64_t gate_rows) {
  if (rows <= 0 || cols <= 0 || gate_rows < 1 || rows % gate_rows) return 0;
  int64_t most = 0;
  for (int form = 0; form < 4; ++form) {
    const NormBwdPlan p = norm_bwd_plan(rows, cols, gate_rows, form & 1, false, form & 2);  // (with a gate: no more workgroups)
    most = std::max(most, 3 * p.groups + (p.strips.strips > 1 ? p.strips.total : 0));
  }
  return 4 * cols * most;
}

extern "C" int mx_residual_norm_bwd(const void* h, int h_f32, const void* r, int r_f32, int64_t rows, int64_t cols,
                                    int64_t ldh, int64_t ldr, const void* post, const void* gate, const void* pre,
                                    int weights_f32, int64_t gate_rows, float scale, const float* rstd, const void* dstream,
                                    const void* dnormed, void* dh, void* dr, void* dpost, void* dgate, void* dpre,
                                    void* workspace, void* stream) {
  if (const int rc = norm_check(h, h_f32, r, r_f32, rows, cols, ldh, ldr, post, gate, pre, weights_f32, gate_rows)) return rc;
  if ((dpost && !post) || (dgate && !gate) || (dpre && !pre) || (dnormed && !pre)) return MX_ERR_INVALID_ARG;
  if (cols == 0) return MX_OK;
  if (rows == 0) return dpost || dgate || dpre ? MX_ERR_INVALID_ARG : MX_OK;
  if (!rstd || !workspace) return MX_ERR_INVALID_ARG;
  auto odd = [](const void* p, int f32) { return ((uintptr_t)p & (f32 ? 3 : 1)) != 0; };
  if (odd(dstream, r_f32) || odd(dnormed, h_f32) || odd(dh, h_f32) || odd(dr, r_f32) || odd(dpost, weights_f32 & 1) ||
      odd(dgate, weights_f32 & 2) || odd(dpre, weights_f32 & 4) || odd(rstd, 1) || ((uintptr_t)workspace & 15))
    return MX_ERR_ALIGNMENT;
  const NormArgs a{h, r, rows, cols, ldh, ldr, {post, weights_f32 & 1}, {gate, weights_f32 & 2}, {pre, weights_f32 & 4},
                   rows / gate_rows, scale, 0.f, norm_past(rows * cols, h_f32, r_f32)};
  const NormBwdPlan plan = norm_bwd_plan(rows, cols, gate_rows, post || gate, gate, a.past);
  const NormStrips s = plan.strips;
  const int64_t groups = plan.groups;
  float* rows_part = (float*)workspace;
  float* gate_part = rows_part + 3 * groups * cols;
  const NormGrads o{dstream, dnormed, dh, dr, rows_part, gate_part, dgate, weights_f32 & 2};
  hipStream_t st = (hipStream_t)stream;
  norm_types(h_f32, r_f32, [&](auto ht, auto rt) {
    using H = decltype(ht);
    using R = decltype(rt);
    norm_shape(cols, [&](auto shape) {
      using S = decltype(shape);
      if constexpr (!norm_shaped<S>)
        hipLaunchKernelGGL((residual_norm_bwd_any_kernel<S::value, H, R>), dim3((unsigned)groups), dim3(S::value), 0, st, a, s, rstd, o);
      else {
        auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(S::kThreads), 0, st, a, s, rstd, o); };
        auto form = [&](auto normed) {
          constexpr bool kNormed = decltype(normed)::value;
          if (!post && !gate) launch(residual_norm_bwd_kernel<S, false, false, kNormed, H, R>);
          else if (!plan.solo) launch(residual_norm_bwd_kernel<S, true, false, kNormed, H, R>);
          else if constexpr (norm_solo_shape<S>()) launch(residual_norm_bwd_kernel<S, true, true, kNormed, H, R>);
        };
        if (dnormed) form(std::true_type());
        else form(std::false_type());
      }
    });
  });
  const int64_t gates = dgate && s.strips > 1 ? gate_rows : 0;  // (fewer than workgroups)
  if (dpost || dpre || gates) {
    const NormJoin j{rows_part, gate_part, groups, s.strips, {dpost, dpre, dgate}, {weights_f32 & 1, weights_f32 & 4, weights_f32 & 2}};
    hipLaunchKernelGGL(residual_norm_join_kernel, dim3((unsigned)((cols + 63) / 64), (unsigned)(2 + gates)), dim3(kNormThreads),
                       0, st, j, cols);
  }
  return hipGetLastError() == hipSuccess ? MX_OK : MX_ERR_LAUNCH;
}
