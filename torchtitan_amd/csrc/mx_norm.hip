// Norms before and after a block, with the block's gate and the residual sum.  For every row of width D, in float32:
//
//   n = h s1 post,  s1 = 1 / sqrt(mean h^2 + eps)       (n = h without a norm behind the block)
//   t = scale r + g n                                    (g n = n without a gate)
//   stream = t,  normed = t s2 pre,  s2 = 1 / sqrt(mean t^2 + eps)
//
// `normed` comes from t before t is rounded to the stream's type.  Backward, from the same h and r (t is formed again:
// as many bytes as reading the stream, without its rounding), with u = normed's gradient times pre:
//
//   e  = dstream + s2 (u - t s2 mean(u t s2)),   dr = scale e,   dpre = sum of rows dnormed t s2
//   dg = sum over the gate's rows of e n,        q = e g
//   dpost = sum of rows q h s1,                  dh = s1 (q post - h s1 mean(q post h s1))
//
// Sums over rows are float32 parts of one workgroup's rows each, joined in order by a second launch: the same result
// on every run.  Row r of T uses row r / (T / G) of a gate of G rows.
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

// Rows of any width, one workgroup a row, element by element; what a later step needs of an earlier one is formed again.
template <class H, class R>
__global__ __launch_bounds__(kNormThreads) void residual_norm_any_kernel(NormArgs a, R* __restrict__ stream,
                                                                         H* __restrict__ normed, float* __restrict__ rstd) {
  __shared__ float part[kNormThreads / 64];
  const int64_t row = blockIdx.x;
  const H* h = (const H*)a.h + row * a.ldh;
  const R* r = (const R*)a.r + row * a.ldr;
  const int64_t g0 = row / a.gate_each * a.cols;
  float s1 = 1.f, s2 = 1.f, sum = 0.f;
  if (a.post.p) {
    for (int64_t c = threadIdx.x; c < a.cols; c += kNormThreads) {
      const float x = norm_element(h + c);
      sum += x * x;
    }
    s1 = 1.f / sqrtf(group_sum<kNormThreads>(sum, part) / (float)a.cols + a.eps);
  }
  auto total = [&](int64_t c) {
    return a.scale * norm_element(r + c) + a.gate.at(g0 + c) * (norm_element(h + c) * s1 * a.post.at(c));
  };
  sum = 0.f;
  for (int64_t c = threadIdx.x; c < a.cols; c += kNormThreads) {
    const float t = total(c);
    stream[row * a.cols + c] = norm_rounded<R>(t);
    sum += t * t;
  }
  if (a.pre.p) {
    s2 = 1.f / sqrtf(group_sum<kNormThreads>(sum, part) / (float)a.cols + a.eps);
    for (int64_t c = threadIdx.x; c < a.cols; c += kNormThreads)
      normed[row * a.cols + c] = norm_rounded<H>(total(c) * s2 * a.pre.at(c));
  }
  if (rstd && threadIdx.x == 0) {
    rstd[row] = s1;
    rstd[a.rows + row] = s2;
  }
}

// How the rows are dealt out in the backward pass: strips of `each` rows that share a row of the gate, `strips` to
// each of its rows; a workgroup takes every gridDim.x-th strip.
struct NormStrips {
  int64_t each, strips, total;
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

template <class H, class R>
__global__ __launch_bounds__(kNormThreads) void residual_norm_bwd_any_kernel(NormArgs a, NormStrips strips,
                                                                             const float* __restrict__ rstd, NormGrads o) {
  __shared__ float part[kNormThreads / 64];
  float* dpost = o.rows_part + (int64_t)blockIdx.x * 3 * a.cols;
  float* dpre = dpost + a.cols;
  float* dgate = o.dgate ? dpre + a.cols : nullptr;
  for (int64_t c = threadIdx.x; c < a.cols; c += kNormThreads) dpost[c] = dpre[c] = 0.f;
  const float width = (float)a.cols;
  for (int64_t strip = blockIdx.x; strip < strips.total; strip += gridDim.x) {
    const int64_t group = strip / strips.strips, part0 = (strip - group * strips.strips) * strips.each;
    const int64_t first = group * a.gate_each + part0;
    const int64_t count = part0 + strips.each < a.gate_each ? strips.each : a.gate_each - part0;
    const int64_t g0 = group * a.cols;
    if (dgate)
      for (int64_t c = threadIdx.x; c < a.cols; c += kNormThreads) dgate[c] = 0.f;
    for (int64_t row = first; row < first + count; ++row) {
      const H* h = (const H*)a.h + row * a.ldh;
      const R* r = (const R*)a.r + row * a.ldr;
      const R* ds = o.dstream ? (const R*)o.dstream + row * a.cols : nullptr;
      const H* dy = o.dnormed ? (const H*)o.dnormed + row * a.cols : nullptr;
      const float s1 = rstd[row], s2 = rstd[a.rows + row];
      auto branch = [&](int64_t c) { return norm_element(h + c) * s1 * a.post.at(c); };
      auto hat = [&](int64_t c) { return (a.scale * norm_element(r + c) + a.gate.at(g0 + c) * branch(c)) * s2; };
      float mean = 0.f;
      if (dy) {
        for (int64_t c = threadIdx.x; c < a.cols; c += kNormThreads) mean += norm_element(dy + c) * a.pre.at(c) * hat(c);
        mean = group_sum<kNormThreads>(mean, part) / width;
      }
      auto inner = [&](int64_t c) {
        const float e = ds ? norm_element(ds + c) : 0.f;
        return dy ? e + s2 * (norm_element(dy + c) * a.pre.at(c) - hat(c) * mean) : e;
      };
      float sum = 0.f;
      for (int64_t c = threadIdx.x; c < a.cols; c += kNormThreads) {
        const float e = inner(c), q = e * a.gate.at(g0 + c), hs = norm_element(h + c) * s1;
        if (o.dr) ((R*)o.dr)[row * a.cols + c] = norm_rounded<R>(a.scale * e);
        if (dy) dpre[c] += norm_element(dy + c) * hat(c);
        if (dgate) dgate[c] += e * branch(c);
        if (a.post.p) dpost[c] += q * hs;
        sum += q * a.post.at(c) * hs;
      }
      if (o.dh) {
        if (a.post.p) sum = group_sum<kNormThreads>(sum, part) / width;
        for (int64_t c = threadIdx.x; c < a.cols; c += kNormThreads) {
          const float q = inner(c) * a.gate.at(g0 + c);
          const float d = a.post.p ? s1 * (q * a.post.at(c) - norm_element(h + c) * s1 * sum) : q;
          ((H*)o.dh)[row * a.cols + c] = norm_rounded<H>(d);
        }
      }
    }
    if (dgate)
      for (int64_t c = threadIdx.x; c < a.cols; c += kNormThreads) {
        if (strips.strips > 1) o.gate_part[strip * a.cols + c] = dgate[c];
        else if (o.dgate_f32) ((float*)o.dgate)[group * a.cols + c] = dgate[c];
        else ((uint16_t*)o.dgate)[group * a.cols + c] = norm_rounded<uint16_t>(dgate[c]);
      }
  }
}

// out[g, c] = sum over the parts p of group g, in order, of part[(g parts + p) stride + c].
__global__ __launch_bounds__(kNormThreads) void residual_norm_join_kernel(const float* __restrict__ part, int64_t parts,
                                                                          int64_t stride, int64_t cols, void* __restrict__ out,
                                                                          int f32) {
  const int64_t c = (int64_t)blockIdx.x * kNormThreads + threadIdx.x, g = blockIdx.y;
  if (c >= cols) return;
  float s = 0.f;
  for (int64_t p = 0; p < parts; ++p) s += part[(g * parts + p) * stride + c];
  if (f32) ((float*)out)[g * cols + c] = s;
  else ((uint16_t*)out)[g * cols + c] = norm_rounded<uint16_t>(s);
}

// Workgroups of the backward pass, and their strips.
constexpr int kNormGroups = 512;

static NormStrips norm_strips(int64_t rows, int64_t gate_rows) {
  const int64_t n = rows / gate_rows;
  int64_t strips = kNormGroups / gate_rows;
  strips = strips < 1 ? 1 : strips > n ? n : strips;
  const int64_t each = (n + strips - 1) / strips;
  strips = (n + each - 1) / each;
  return {each, strips, strips * gate_rows};
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
  if (rows > 0x7FFFFFFF || cols > 0x7FFFFFFF) return MX_ERR_UNSUPPORTED;
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
                   rows / gate_rows, scale, eps};
  norm_types(h_f32, r_f32, [&](auto ht, auto rt) {
    using H = decltype(ht);
    using R = decltype(rt);
    hipLaunchKernelGGL((residual_norm_any_kernel<H, R>), dim3((unsigned)rows), dim3(kNormThreads), 0, (hipStream_t)stream, a,
                       (R*)stream_out, (H*)normed, rstd);
  });
  return hipGetLastError() == hipSuccess ? MX_OK : MX_ERR_LAUNCH;
}

extern "C" int64_t mx_residual_norm_workspace(int64_t rows, int64_t cols, int64_t gate_rows) {
  if (rows <= 0 || cols <= 0 || gate_rows < 1 || rows % gate_rows) return 0;
  const NormStrips s = norm_strips(rows, gate_rows);
  const int64_t groups = s.total < kNormGroups ? s.total : kNormGroups;
  return 4 * cols * (3 * groups + (s.strips > 1 ? s.total : 0));
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
                   rows / gate_rows, scale, 0.f};
  const NormStrips s = norm_strips(rows, gate_rows);
  const int64_t groups = s.total < kNormGroups ? s.total : kNormGroups;
  float* rows_part = (float*)workspace;
  float* gate_part = rows_part + 3 * groups * cols;
  const NormGrads o{dstream, dnormed, dh, dr, rows_part, gate_part, dgate, weights_f32 & 2};
  hipStream_t st = (hipStream_t)stream;
  norm_types(h_f32, r_f32, [&](auto ht, auto rt) {
    hipLaunchKernelGGL((residual_norm_bwd_any_kernel<decltype(ht), decltype(rt)>), dim3((unsigned)groups), dim3(kNormThreads),
                       0, st, a, s, rstd, o);
  });
  const unsigned blocks = (unsigned)((cols + kNormThreads - 1) / kNormThreads);
  auto join = [&](void* out, const float* part, int64_t parts, int64_t stride, int64_t many, int f32) {
    for (int64_t g = 0; out && g < many; g += 65535) {  // (a grid has at most as many rows)
      const int64_t now = many - g < 65535 ? many - g : 65535;
      hipLaunchKernelGGL(residual_norm_join_kernel, dim3(blocks, (unsigned)now), dim3(kNormThreads), 0, st,
                         part + g * parts * stride, parts, stride, cols,
                         f32 ? (void*)((float*)out + g * cols) : (void*)((uint16_t*)out + g * cols), f32);
    }
  };
  join(dpost, rows_part, groups, 3 * cols, 1, weights_f32 & 1);
  join(dpre, rows_part + cols, groups, 3 * cols, 1, weights_f32 & 4);
  if (s.strips > 1) join(dgate, gate_part, s.strips, cols, gate_rows, weights_f32 & 2);
  return hipGetLastError() == hipSuccess ? MX_OK : MX_ERR_LAUNCH;
}
