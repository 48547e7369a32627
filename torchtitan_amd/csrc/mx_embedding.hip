// Token embedding and its gradient.
//
//   out[t, :]  = scale * W[id(t) - first, :]                  (zeros where that row is not in the table)
//   dW[v, :]   = scale * sum over t with id(t) - first = v, id(t) != padding, of dout[t, :]
//
// Both are bound by memory.  The gradient writes every row of the table, zeros where no token asked for it, and is the
// same on every run: equal ids are summed in the order of their tokens, in float32, and rounded once.
#include "mx_rows.h"

namespace mx {

constexpr int kEmbThreads = 256;
constexpr int kEmbWaves = kEmbThreads / 64;

struct EmbIds {
  const void* ids;
  int wide;  // int64, else int32
  int64_t first, rows, padding;
  // Row of token t in the table, or `rows` for one that is not in it.
  __device__ __forceinline__ uint32_t row(int64_t t) const {
    const int64_t id = wide ? ((const int64_t*)ids)[t] : (int64_t)((const int32_t*)ids)[t];
    // (unsigned: an id below the first wraps to a number that no table has)
    const uint64_t r = (uint64_t)id - (uint64_t)first;
    return r < (uint64_t)rows ? (uint32_t)r : (uint32_t)rows;
  }
  __device__ __forceinline__ uint32_t key(int64_t t) const {
    const int64_t id = wide ? ((const int64_t*)ids)[t] : (int64_t)((const int32_t*)ids)[t];
    return id == padding ? (uint32_t)rows : row(t);
  }
};

// One wave a token: the row's pieces are asked for four at a time.
template <class W, class O>
__global__ __launch_bounds__(kEmbThreads) void embedding_kernel(EmbIds ids, int64_t n, const W* __restrict__ weight,
                                                                int64_t cols, int64_t ldw, float scale,
                                                                O* __restrict__ out) {
  constexpr int V = 8, U = 4;
  const int64_t t = (int64_t)blockIdx.x * kEmbWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (t >= n) return;
  const uint32_t r = __builtin_amdgcn_readfirstlane(ids.row(t));
  const bool in = r < (uint32_t)ids.rows;
  const W* src = weight + (in ? (int64_t)r * ldw : 0);
  O* dst = out + t * cols;
  for (int64_t c0 = (int64_t)(threadIdx.x & 63) * V; c0 < cols; c0 += 64 * V * U) {
    Piece<W, V> p[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t c = c0 + u * 64 * V;
      if (in) load_piece<false>(src + c, cols - c, p[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t c = c0 + u * 64 * V;
      float f[V] = {};
      if (in) {
        to_floats(p[u], f);
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] *= scale;
      }
      store_piece<false>(dst + c, cols - c, from_floats<O>(f));
    }
  }
}

// Stable order of the tokens by their rows: a token's place is the number of tokens with a smaller row, or with its
// row and in front of it.  A workgroup places 64 tokens; every wave counts over a sixteenth of the tokens.
constexpr int kRankThreads = 1024, kRankTile = 8192;

__global__ __launch_bounds__(kRankThreads) void embedding_rank_kernel(EmbIds ids, int64_t n, uint32_t* __restrict__ keys,
                                                                      uint32_t* __restrict__ places) {
  __shared__ uint32_t tile[kRankTile];
  __shared__ uint32_t counts[kRankThreads / 64][64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t t = (int64_t)blockIdx.x * 64 + lane;
  const uint32_t mine = t < n ? ids.key(t) : 0xFFFFFFFFu;
  uint32_t before = 0;
  for (int64_t base = 0; base < n; base += kRankTile) {
    const int m = (int)(n - base < kRankTile ? n - base : kRankTile);
    __syncthreads();
    for (int i = threadIdx.x; i < m; i += kRankThreads) tile[i] = ids.key(base + i);
    __syncthreads();
    const int each = (m + 15) / 16, lo = wave * each, hi = lo + each < m ? lo + each : m;
    for (int i = lo; i < hi; ++i) {
      const uint32_t k = tile[i];
      before += k < mine || (k == mine && base + i < t);
    }
  }
  counts[wave][lane] = before;
  __syncthreads();
  if (wave == 0 && t < n) {
    uint32_t at = 0;
    for (int w = 0; w < kRankThreads / 64; ++w) at += counts[w][lane];
    keys[at] = mine;
    places[at] = (uint32_t)t;
  }
}

__device__ __forceinline__ int64_t emb_lower_bound(const uint32_t* __restrict__ keys, int64_t n, uint32_t key) {
  int64_t lo = 0, hi = n;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (keys[mid] < key) lo = mid + 1; else hi = mid;
  }
  return lo;
}

// One wave a row of the table: its tokens' gradients, found by a search in the sorted rows, summed in order.
template <class D, class G>
__global__ __launch_bounds__(kEmbThreads) void embedding_grad_kernel(const D* __restrict__ dout, int64_t n, int64_t ldd,
                                                                     const uint32_t* __restrict__ keys,
                                                                     const uint32_t* __restrict__ places, int64_t rows,
                                                                     int64_t cols, float scale, G* __restrict__ grad) {
  constexpr int V = 8;
  const int64_t v = (int64_t)blockIdx.x * kEmbWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (v >= rows) return;
  const int64_t lo = emb_lower_bound(keys, n, (uint32_t)v), hi = emb_lower_bound(keys, n, (uint32_t)v + 1);
  for (int64_t c = (int64_t)(threadIdx.x & 63) * V; c < cols; c += 64 * V) {
    float acc[V] = {};
    for (int64_t i = lo; i < hi; ++i) {
      Piece<D, V> p;
      load_piece<false>(dout + (int64_t)places[i] * ldd + c, cols - c, p);
      float f[V];
      to_floats(p, f);
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] += f[e];
    }
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] *= scale;
    store_piece<false>(grad + v * cols + c, cols - c, from_floats<G>(acc));
  }
}

// Calls f(T()) with T the element type that the flag names.
template <class F>
static auto of_type(int f32, F&& f) {
  return f32 ? f(float()) : f(uint16_t());
}

}  // namespace mx

using namespace mx;

extern "C" int mx_embedding(const void* ids, int ids_i64, int64_t n, const void* weight, int weight_f32, int64_t rows,
                            int64_t cols, int64_t ldw, int64_t first, float scale, void* out, int out_f32, void* stream) {
  if (n < 0 || rows < 0 || cols < 0 || (rows > 1 && ldw < cols)) return MX_ERR_INVALID_ARG;
  if (n == 0 || cols == 0) return MX_OK;
  if (!ids || (rows > 0 && !weight) || !out) return MX_ERR_INVALID_ARG;
  const uintptr_t w_odd = weight_f32 ? 3 : 1, o_odd = out_f32 ? 3 : 1;
  if (((uintptr_t)ids & (ids_i64 ? 7 : 3)) || ((uintptr_t)weight & w_odd) || ((uintptr_t)out & o_odd)) return MX_ERR_ALIGNMENT;
  const int64_t groups = (n + kEmbWaves - 1) / kEmbWaves;
  if (rows >= 0x7FFFFFFF || groups > 0x7FFFFFFF) return MX_ERR_UNSUPPORTED;
  const EmbIds e{ids, ids_i64 != 0, first, rows, 0};
  of_type(weight_f32, [&](auto w) {
    of_type(out_f32, [&](auto o) {
      hipLaunchKernelGGL((embedding_kernel<decltype(w), decltype(o)>), dim3((unsigned)groups), dim3(kEmbThreads), 0,
                         (hipStream_t)stream, e, n, (const decltype(w)*)weight, cols, ldw, scale, (decltype(o)*)out);
    });
  });
  return hipGetLastError() == hipSuccess ? MX_OK : MX_ERR_LAUNCH;
}

extern "C" int64_t mx_embedding_grad_workspace(int64_t n, int64_t rows, int64_t cols) {
  if (n <= 0 || rows <= 0 || cols <= 0) return 0;
  return 8 * n;
}

extern "C" int mx_embedding_grad(const void* ids, int ids_i64, int64_t n, const void* dout, int dout_f32, int64_t ldd,
                                 int64_t rows, int64_t cols, int64_t first, int64_t padding, float scale, void* grad,
                                 int grad_f32, void* workspace, void* stream) {
  if (n < 0 || rows < 0 || cols < 0 || (n > 1 && ldd < cols)) return MX_ERR_INVALID_ARG;
  if (rows == 0 || cols == 0) return MX_OK;
  if (!grad || (n > 0 && (!ids || !dout || !workspace))) return MX_ERR_INVALID_ARG;
  const uintptr_t d_odd = dout_f32 ? 3 : 1, g_odd = grad_f32 ? 3 : 1;
  if (((uintptr_t)ids & (ids_i64 ? 7 : 3)) || ((uintptr_t)dout & d_odd) || ((uintptr_t)grad & g_odd) ||
      ((uintptr_t)workspace & 15))
    return MX_ERR_ALIGNMENT;
  if (rows >= 0x7FFFFFFF || n >= 0x7FFFFFFF) return MX_ERR_UNSUPPORTED;
  hipStream_t st = (hipStream_t)stream;
  uint32_t* keys = (uint32_t*)workspace;
  uint32_t* places = keys + n;
  const EmbIds e{ids, ids_i64 != 0, first, rows, padding};
  if (n > 0)
    hipLaunchKernelGGL(embedding_rank_kernel, dim3((unsigned)((n + 63) / 64)), dim3(kRankThreads), 0, st, e, n, keys, places);
  of_type(dout_f32, [&](auto d) {
    of_type(grad_f32, [&](auto g) {
      hipLaunchKernelGGL((embedding_grad_kernel<decltype(d), decltype(g)>), dim3((unsigned)((rows + kEmbWaves - 1) / kEmbWaves)),
                         dim3(kEmbThreads), 0, st, (const decltype(d)*)dout, n, ldd, keys, places, rows, cols, scale,
                         (decltype(g)*)grad);
    });
  });
  return hipGetLastError() == hipSuccess ? MX_OK : MX_ERR_LAUNCH;
}
