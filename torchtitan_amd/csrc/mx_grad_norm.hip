// The norm of all gradients of a model taken as one vector, and their scaling to a limit.
//
//   N = sqrt(sum g^2)  or  sum |g|  or  max |g|          g *= f,  f = min(1, limit / (N + 1e-6))
//
// Bound by memory: every gradient is read for the norm and, where f is below 1, read and written once more.  Squares
// and sums are held in 64 bits: their order does not matter to the result's 32, and gradients of 1e-25 or 1e25 keep
// their norm.  A table of tensors travels as a kernel argument; a tensor is cut into chunks, a workgroup takes every
// gridDim.x-th chunk of its launch and leaves one part, and whoever needs the norm joins the parts in order.
#include <algorithm>
#include <vector>

#include "mx_rows.h"

namespace mx {

constexpr int kGradThreads = 256;
constexpr int kGradPieces = 4;                                   // 16-byte pieces a lane and chunk
constexpr int64_t kGradChunk = 16 * kGradThreads * kGradPieces;  // bytes
constexpr int kGradTensors = 160;                                // of one launch
constexpr int kGradGroups = 1536;                                // workgroups of one launch (but see GradFactor)

struct GradEntry {
  void* p;
  int64_t elems;
  uint32_t first;  // first chunk of this tensor
  uint32_t f32;
};
struct GradTable {
  GradEntry e[kGradTensors];
};

__device__ __forceinline__ int grad_find(const GradTable& t, int n, uint32_t chunk) {
  int lo = 0, hi = n;  // the last entry whose first chunk is not behind this one
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.e[mid].first <= chunk) lo = mid; else hi = mid;
  }
  return lo;
}

enum { kGradTwo = 0, kGradOne = 1, kGradMax = 2 };

// NaN is not lost in a maximum: it stays the answer once it is there.
__device__ __forceinline__ double grad_max(double a, double b) { return a != a || a > b ? a : b; }
template <int KIND>
__device__ __forceinline__ double grad_join(double a, double b) {
  return KIND == kGradMax ? grad_max(a, b) : a + b;
}
template <int KIND>
__device__ __forceinline__ double grad_add(double acc, float x) {
  const double d = (double)x;
  if (KIND == kGradTwo) return __builtin_fma(d, d, acc);
  return grad_join<KIND>(acc, __builtin_fabs(d));
}
template <int KIND>
__device__ __forceinline__ double grad_group_join(double v, double* part) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = grad_join<KIND>(v, __shfl_xor(v, off, 64));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = part[0];
#pragma unroll
  for (int w = 1; w < kGradThreads / 64; ++w) v = grad_join<KIND>(v, part[w]);
  return v;
}

template <int KIND, class T>
__device__ __forceinline__ double grad_chunk(const T* p, int64_t left, double acc) {
  constexpr int V = 16 / sizeof(T);
  Piece<T, V> q[kGradPieces];
#pragma unroll
  for (int k = 0; k < kGradPieces; ++k) {
    const int64_t at = (int64_t)(k * kGradThreads + threadIdx.x) * V;
    load_piece<true>(p + at, left - at, q[k]);
  }
#pragma unroll
  for (int k = 0; k < kGradPieces; ++k) {
    float f[V];
    to_floats(q[k], f);
#pragma unroll
    for (int e = 0; e < V; ++e) acc = grad_add<KIND>(acc, f[e]);
  }
  return acc;
}

template <int KIND>
__global__ __launch_bounds__(kGradThreads) void grad_norm_kernel(GradTable table, int n, uint32_t chunks,
                                                                 double* __restrict__ parts) {
  __shared__ double part[kGradThreads / 64];
  double acc = 0.0;
  for (uint32_t chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    const GradEntry e = table.e[grad_find(table, n, chunk)];
    const int64_t at = (int64_t)(chunk - e.first) * (kGradChunk / (e.f32 ? 4 : 2));
    if (e.f32) acc = grad_chunk<KIND>((const float*)e.p + at, e.elems - at, acc);
    else acc = grad_chunk<KIND>((const uint16_t*)e.p + at, e.elems - at, acc);
  }
  acc = grad_group_join<KIND>(acc, part);
  if (threadIdx.x == 0) parts[blockIdx.x] = acc;
}

// The norm from its parts, in every lane of the workgroup.
template <int KIND>
__device__ __forceinline__ float grad_joined(const double* __restrict__ parts, int64_t n, double* part) {
  double acc = 0.0;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < n; i += kGradThreads) acc = grad_join<KIND>(acc, parts[i]);
  acc = grad_group_join<KIND>(acc, part);
  return (float)(KIND == kGradTwo ? __builtin_sqrt(acc) : acc);
}
template <int KIND>
__global__ __launch_bounds__(kGradThreads) void grad_norm_join_kernel(const double* __restrict__ parts, int64_t n,
                                                                      float* __restrict__ norm) {
  __shared__ double part[kGradThreads / 64];
  const float all = grad_joined<KIND>(parts, n, part);
  if (threadIdx.x == 0) *norm = all;
}

template <class T>
__device__ __forceinline__ void grad_scale_chunk(T* p, int64_t left, float f) {
  constexpr int V = 16 / sizeof(T);
  Piece<T, V> q[kGradPieces];
#pragma unroll
  for (int k = 0; k < kGradPieces; ++k) {
    const int64_t at = (int64_t)(k * kGradThreads + threadIdx.x) * V;
    load_piece<true>(p + at, left - at, q[k]);
  }
#pragma unroll
  for (int k = 0; k < kGradPieces; ++k) {
    const int64_t at = (int64_t)(k * kGradThreads + threadIdx.x) * V;
    float v[V];
    to_floats(q[k], v);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] *= f;
    store_piece<true>(p + at, left - at, from_floats<T>(v));
  }
}

// f from the norm, or (count > 0) from its parts, joined here by every workgroup: one launch less.  A factor of exactly 1
// leaves every gradient as it is: nothing is read.  Chunks are taken from the last to the first: what the norm has read
// last is still in the last cache.  A workgroup for every chunk, so that the chip works its way through memory in order:
// 3.3 GB of float32 1092 us, where 2048 workgroups that come back for more take 1253; but those do where each joins
// the parts.
struct GradFactor {
  const double* parts;
  int64_t count;
  float* norm;  // read, or (count > 0) written
  float limit;
};
template <int KIND>
__global__ __launch_bounds__(kGradThreads) void grad_scale_kernel(GradTable table, int n, uint32_t chunks, GradFactor by) {
  __shared__ double part[kGradThreads / 64];
  float norm;
  if (by.count > 0) {
    norm = grad_joined<KIND>(by.parts, by.count, part);
    if (blockIdx.x == 0 && threadIdx.x == 0) *by.norm = norm;
  } else {
    norm = *by.norm;
  }
  const float f0 = by.limit / (norm + 1e-6f), f = f0 > 1.f ? 1.f : f0;  // (NaN stays)
  if (f == 1.f) return;
  for (uint32_t i = blockIdx.x; i < chunks; i += gridDim.x) {
    const uint32_t chunk = chunks - 1 - i;
    const GradEntry e = table.e[grad_find(table, n, chunk)];
    const int64_t at = (int64_t)(chunk - e.first) * (kGradChunk / (e.f32 ? 4 : 2));
    if (e.f32) grad_scale_chunk((float*)e.p + at, e.elems - at, f);
    else grad_scale_chunk((uint16_t*)e.p + at, e.elems - at, f);
  }
}

static int64_t grad_chunks(int64_t elems, int f32) {
  const int64_t per = kGradChunk / (f32 ? 4 : 2);
  return (elems + per - 1) / per;
}

static int grad_check(int64_t n, void* const* p, const int64_t* elems, const int32_t* is_f32) {
  if (n < 0 || (n > 0 && (!p || !elems || !is_f32))) return MX_ERR_INVALID_ARG;
  int64_t chunks = 0;
  for (int64_t i = 0; i < n; ++i) {
    if (elems[i] < 0 || (elems[i] > 0 && !p[i])) return MX_ERR_INVALID_ARG;
    if ((uintptr_t)p[i] & (is_f32[i] ? 3 : 1)) return MX_ERR_ALIGNMENT;
    // (a workgroup each, and a launch has fewer than 2^32 lanes: 256 GB)
    if ((chunks += grad_chunks(elems[i], is_f32[i])) > 0xFFFFFF) return MX_ERR_UNSUPPORTED;
  }
  return MX_OK;
}

// Whether two of the tensors share memory (where that cannot be found out: yes, the slower answer).
static bool grad_overlap(int64_t n, void* const* p, const int64_t* elems, const int32_t* is_f32) try {
  std::vector<std::pair<uintptr_t, uintptr_t>> runs;
  runs.reserve(n);
  for (int64_t i = 0; i < n; ++i)
    if (elems[i]) runs.emplace_back((uintptr_t)p[i], (uintptr_t)p[i] + elems[i] * (is_f32[i] ? 4 : 2));
  std::sort(runs.begin(), runs.end());
  for (size_t i = 1; i < runs.size(); ++i)
    if (runs[i].first < runs[i - 1].second) return true;
  return false;
} catch (...) {
  return true;
}

// Tables of up to `most` non-empty tensors, each handed to launch(table, tensors, chunks).
template <class Launch>
static int grad_launches(int64_t n, void* const* p, const int64_t* elems, const int32_t* is_f32, int most, Launch&& launch) {
  GradTable table;
  int used = 0;
  int64_t chunks = 0;
  auto flush = [&]() -> int {
    if (used == 0) return MX_OK;
    launch(table, used, (uint32_t)chunks);
    used = 0;
    chunks = 0;
    return hipGetLastError() == hipSuccess ? MX_OK : MX_ERR_LAUNCH;
  };
  for (int64_t i = 0; i < n; ++i) {
    if (elems[i] == 0) continue;
    const int64_t mine = grad_chunks(elems[i], is_f32[i]);
    if (used == most)
      if (const int rc = flush()) return rc;
    table.e[used++] = {p[i], elems[i], (uint32_t)chunks, is_f32[i] != 0};
    chunks += mine;
  }
  return flush();
}

static unsigned grad_groups(uint32_t chunks) { return chunks < kGradGroups ? chunks : kGradGroups; }

template <class F>
static int grad_kind(int kind, F&& f) {
  switch (kind) {
    case kGradTwo: return f(std::integral_constant<int, kGradTwo>());
    case kGradOne: return f(std::integral_constant<int, kGradOne>());
    default: return f(std::integral_constant<int, kGradMax>());
  }
}

}  // namespace mx

using namespace mx;

extern "C" int64_t mx_grad_norm_workspace(int64_t n) {
  return n <= 0 ? 0 : 8 * kGradGroups * ((n + kGradTensors - 1) / kGradTensors);
}

// The parts of the norm in `parts`, how many in `count`.
template <int KIND>
static int grad_parts(int64_t n, void* const* grads, const int64_t* elems, const int32_t* is_f32, double* parts, int64_t& count,
                      hipStream_t st) {
  count = 0;
  return grad_launches(n, grads, elems, is_f32, kGradTensors, [&](const GradTable& t, int m, uint32_t chunks) {
    const unsigned groups = grad_groups(chunks);
    hipLaunchKernelGGL(grad_norm_kernel<KIND>, dim3(groups), dim3(kGradThreads), 0, st, t, m, chunks, parts + count);
    count += groups;
  });
}

template <int KIND>
static int grad_joined_launch(const double* parts, int64_t count, float* norm, hipStream_t st) {
  hipLaunchKernelGGL(grad_norm_join_kernel<KIND>, dim3(1), dim3(kGradThreads), 0, st, parts, count, norm);
  return hipGetLastError() == hipSuccess ? MX_OK : MX_ERR_LAUNCH;
}

template <int KIND>
static int grad_scaled(int64_t n, void* const* grads, const int64_t* elems, const int32_t* is_f32, const GradFactor& by,
                       hipStream_t st) {
  // tensors that share memory are scaled one after the other, as a loop over them would
  const int most = grad_overlap(n, grads, elems, is_f32) ? 1 : kGradTensors;
  return grad_launches(n, grads, elems, is_f32, most, [&](const GradTable& t, int m, uint32_t chunks) {
    hipLaunchKernelGGL(grad_scale_kernel<KIND>, dim3(by.count > 0 ? grad_groups(chunks) : chunks), dim3(kGradThreads), 0, st, t,
                       m, chunks, by);
  });
}

static int grad_norm_check(int64_t n, void* const* grads, const int64_t* elems, const int32_t* is_f32, int kind,
                           const float* norm, const void* workspace) {
  if (const int rc = grad_check(n, grads, elems, is_f32)) return rc;
  if (kind < kGradTwo || kind > kGradMax || !norm || (n > 0 && !workspace)) return MX_ERR_INVALID_ARG;
  return ((uintptr_t)norm & 3) || ((uintptr_t)workspace & 7) ? MX_ERR_ALIGNMENT : MX_OK;
}

extern "C" int mx_grad_norm(int64_t n, void* const* grads, const int64_t* elems, const int32_t* is_f32, int kind, float* norm,
                            void* workspace, void* stream) {
  if (const int rc = grad_norm_check(n, grads, elems, is_f32, kind, norm, workspace)) return rc;
  return grad_kind(kind, [&](auto k) {
    constexpr int K = decltype(k)::value;
    int64_t count;
    if (const int rc = grad_parts<K>(n, grads, elems, is_f32, (double*)workspace, count, (hipStream_t)stream)) return rc;
    return grad_joined_launch<K>((const double*)workspace, count, norm, (hipStream_t)stream);
  });
}

extern "C" int mx_grad_scale(int64_t n, void* const* grads, const int64_t* elems, const int32_t* is_f32, const float* norm,
                             float limit, void* stream) {
  if (const int rc = grad_check(n, grads, elems, is_f32)) return rc;
  if (!norm) return MX_ERR_INVALID_ARG;
  if ((uintptr_t)norm & 3) return MX_ERR_ALIGNMENT;
  return grad_scaled<kGradTwo>(n, grads, elems, is_f32, {nullptr, 0, const_cast<float*>(norm), limit}, (hipStream_t)stream);
}

extern "C" int mx_grad_clip(int64_t n, void* const* grads, const int64_t* elems, const int32_t* is_f32, int kind, float* norm,
                            float limit, void* workspace, void* stream) {
  if (const int rc = grad_norm_check(n, grads, elems, is_f32, kind, norm, workspace)) return rc;
  hipStream_t st = (hipStream_t)stream;
  return grad_kind(kind, [&](auto k) {
    constexpr int K = decltype(k)::value;
    const double* parts = (const double*)workspace;
    int64_t count;
    if (const int rc = grad_parts<K>(n, grads, elems, is_f32, (double*)workspace, count, st)) return rc;
    // Above half a gigabyte the parts are joined once, for workgroups that take one chunk each (and with no parts, where all
    // tensors are empty, nobody else writes the norm).  100 MB: 34.6 us without, 34.2 and the join's 4 with.
    int64_t chunks = 0;
    for (int64_t i = 0; i < n; ++i) chunks += grad_chunks(elems[i], is_f32[i]);
    if (count == 0 || chunks * kGradChunk > (int64_t{512} << 20)) {
      if (const int rc = grad_joined_launch<K>(parts, count, norm, st)) return rc;
      count = 0;
    }
    return grad_scaled<K>(n, grads, elems, is_f32, {parts, count, norm, limit}, st);
  });
}
