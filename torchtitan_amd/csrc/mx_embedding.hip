// Token embedding and its gradient.
//
//   out[t, :]  = scale * W[id(t) - first, :]                  (zeros where that row is not in the table)
//   dW[v, :]   = scale * sum over t with id(t) - first = v, id(t) != padding, of dout[t, :]
//
// Both are bound by memory.  The gradient writes every row of the table, zeros where no token asked for it: the tokens
// are put in order by their rows, and every run of equal rows is summed in float32 and rounded once.  Which sums are
// formed of a row depends on its own tokens and the number of all tokens alone, so the gradient is the same on every
// run, and that of a part of the table the same as those rows of the whole's.
#include <algorithm>

#include "mx_rows.h"

namespace mx {

constexpr int kEmbThreads = 256;
constexpr int kEmbWaves = kEmbThreads / 64;
constexpr int64_t kEmbGroups = 0xFFFFFF;  // workgroups of at most 256 lanes: a launch has fewer than 2^32 lanes

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

// Wider rows: one wave for 1024 columns of a token, all asked for before the first is stored: 147456 x 2048 151 us (604 MB written and
// as many read, most of them from the caches; with 2048 columns a wave 156), 8192 x 4096 of a shard 18 (with a wave for the
// whole row 24).
constexpr int kEmbPieces = 2, kEmbSlab = 64 * 8 * kEmbPieces;
template <class W, class O>
__global__ __launch_bounds__(kEmbThreads) void embedding_kernel(EmbIds ids, int64_t n, const W* __restrict__ weight,
                                                                int64_t cols, int64_t ldw, float scale, bool past, uint32_t slabs,
                                                                O* __restrict__ out) {
  constexpr int V = 8, U = kEmbPieces;
  const uint32_t item = blockIdx.x * (uint32_t)kEmbWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), t = item / slabs;
  if (t >= n) return;
  const uint32_t r = __builtin_amdgcn_readfirstlane(ids.row(t));
  const bool in = r < (uint32_t)ids.rows;
  const int64_t c0 = (int64_t)(item - t * slabs) * kEmbSlab + (threadIdx.x & 63) * V;
  const W* src = weight + (in ? (int64_t)r * ldw : 0);
  O* dst = out + (int64_t)t * cols;
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
    const Piece<O, V> q = from_floats<O>(f);
    if (past) store_piece<true>(dst + c, cols - c, q);
    else store_piece<false>(dst + c, cols - c, q);
  }
}

// Rows of up to 512 columns: 8 to 64 lanes (1 << shift) a token, a piece each, two tokens a lane.  us for a million tokens, with a
// wave for each / so: 512 columns 290 / 272, 256 254 / 134, 64 259 / 34.
constexpr int kEmbTokens = 2;
template <class W, class O>
__global__ __launch_bounds__(kEmbThreads) void embedding_narrow_kernel(EmbIds ids, int64_t n, const W* __restrict__ weight,
                                                                       int64_t cols, int64_t ldw, float scale, bool past, int shift,
                                                                       O* __restrict__ out) {
  constexpr int V = 8;
  const int64_t c = (int64_t)(threadIdx.x & ((1 << shift) - 1)) * V, left = cols - c;
  const int64_t step = kEmbThreads >> shift, t0 = (int64_t)blockIdx.x * step * kEmbTokens + (threadIdx.x >> shift);
  uint32_t r[kEmbTokens];
#pragma unroll
  for (int k = 0; k < kEmbTokens; ++k) r[k] = t0 + k * step < n ? ids.row(t0 + k * step) : (uint32_t)ids.rows;
  Piece<W, V> p[kEmbTokens];
#pragma unroll
  for (int k = 0; k < kEmbTokens; ++k) load_piece<false>(weight + (int64_t)r[k] * ldw + c, r[k] < (uint32_t)ids.rows ? left : 0, p[k]);
#pragma unroll
  for (int k = 0; k < kEmbTokens; ++k) {
    if (t0 + k * step >= n) break;
    float f[V];
    to_floats(p[k], f);
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = r[k] < (uint32_t)ids.rows ? f[e] * scale : 0.f;
    const Piece<O, V> q = from_floats<O>(f);
    O* dst = out + (t0 + k * step) * cols + c;
    if (past) store_piece<true>(dst, left, q);
    else store_piece<false>(dst, left, q);
  }
}

// ---- work that rides along in the launches that sort, whose own work leaves most of the chip idle: workgroups behind the
// first `own` write zeros, 16 bytes a lane, in the order of memory (6.3 TB/s; workgroups that each go through a part of
// their own reach 5.2).  Either all of a piece of memory (rows that tokens have are written over
// later), or the rows of the gradient that no token has, by the flags that an earlier launch has set.
enum { kRideFill = 0, kRideMark = 1, kRideUnused = 2 };
struct EmbRide {
  int mode;
  unsigned own;    // workgroups of the launch's own work
  uint8_t* to;     // memory to fill, the flags to set, or the gradient
  int64_t count;   // bytes, tokens, or 16-byte pieces of rows from piece `from` on
  bool past;       // the gradient does not stay in the last cache: stored past it
  EmbIds ids;
  const uint8_t* used;  // a flag a row
  int64_t from, row_bytes;
};

__device__ __forceinline__ void store_zeros(uint8_t* to, int64_t bytes, bool past) {
  const Piece<uint16_t, 8> zero{};
  if (past) store_piece<true>((uint16_t*)to, bytes / 2, zero);
  else store_piece<false>((uint16_t*)to, bytes / 2, zero);
}

// Whether the calling workgroup of THREADS lanes has ridden along (and is done).
template <int THREADS>
__device__ __forceinline__ bool rode(const EmbRide& q) {
  if (blockIdx.x < q.own) return false;
  const int64_t base = (int64_t)(blockIdx.x - q.own) * THREADS, i = base + threadIdx.x;
  if (q.mode == kRideFill) {
    store_zeros(q.to + i * 16, q.count - i * 16, q.past);
  } else if (i < q.count) {
    if (q.mode == kRideMark) {
      const uint32_t r = q.ids.key(i);
      if (r < (uint32_t)q.ids.rows) q.to[r] = 1;  // (whoever sets a flag sets it to 1)
    } else {
      // one division of long numbers a workgroup, a short one for its lanes
      const uint32_t each = (uint32_t)((q.row_bytes + 15) / 16);
      const int64_t row0 = (q.from + base) / each;
      const uint32_t piece = (uint32_t)(q.from + base - row0 * each) + threadIdx.x, r = piece / each;
      const int64_t c = (int64_t)(piece - r * each) * 16;
      if (!q.used[row0 + r]) store_zeros(q.to + (row0 + r) * q.row_bytes + c, q.row_bytes - c, q.past);
    }
  }
  return true;
}
static int64_t ride_groups(int64_t pieces, int threads) { return (pieces + threads - 1) / threads; }

__global__ __launch_bounds__(256) void embedding_zeros_kernel(EmbRide ride) { rode<256>(ride); }

// ---- the order of the tokens by their rows, stable: up to kRankMost tokens in one launch, more by radix passes

// A token's place is the number of tokens with a smaller row, or with its row and in front of it.  A workgroup places
// kRankThreads / parts tokens: every one is held by `parts` lanes, which count over a share of all tokens each, four rows
// a read of LDS.  Two instructions a pair; parts so that there is a workgroup for every CU: 2003 tokens 5.9 us, 8192 16.6,
// where two radix passes take 33.
constexpr int kRankThreads = 1024, kRankMost = 8192, kRankKeys = kRankMost + 4 * kRankThreads / 8;

// Tokens of a workgroup, and how many rows a lane compares with: an odd number of fours, so that the shares of lanes
// next to each other begin in different banks.
static int rank_tokens(int64_t n) { return n > 4096 ? 32 : n > 2048 ? 16 : 8; }
__host__ __device__ inline int rank_share(int n, int parts) {
  const int fours = (n + 4 * parts - 1) / (4 * parts);
  return 4 * (fours | 1);
}

__global__ __launch_bounds__(kRankThreads) void embedding_rank_kernel(EmbIds ids, int n, int tokens, uint32_t* __restrict__ keys,
                                                                      uint32_t* __restrict__ places,
                                                                      uint32_t* __restrict__ chains, EmbRide ride) {
  if (rode<kRankThreads>(ride)) return;
  __shared__ alignas(16) uint32_t tile[kRankKeys];
  __shared__ uint32_t counts[kRankThreads];
  const int parts = kRankThreads / tokens, share = rank_share(n, parts);
  const int part = threadIdx.x / tokens, at = threadIdx.x % tokens, t0 = (int)blockIdx.x * tokens, t = t0 + at;
  if (blockIdx.x == 0 && threadIdx.x == 0) *chains = 0;
  uint32_t own[kRankMost / kRankThreads];  // (all asked for before the first is written)
#pragma unroll
  for (int k = 0; k < kRankMost / kRankThreads; ++k) {
    const int i = k * kRankThreads + threadIdx.x;
    own[k] = i < n ? ids.key(i) : 0xFFFFFFFFu;  // (in front of nobody)
  }
#pragma unroll
  for (int k = 0; k < kRankMost / kRankThreads; ++k) tile[k * kRankThreads + threadIdx.x] = own[k];
  for (int i = kRankMost + threadIdx.x; i < kRankKeys; i += kRankThreads) tile[i] = 0xFFFFFFFFu;
  __syncthreads();
  const uint32_t mine = t < n ? tile[t] : 0u;
  const int lo = part * share, hi = lo + share;
  uint32_t before = 0;
  auto count = [&](auto&& limit) {
#pragma unroll 4
    for (int i = lo; i < hi; i += 4) {
      const u32x4 k = *reinterpret_cast<const u32x4*>(tile + i);
      before += k.x < limit(i);
      before += k.y < limit(i + 1);
      before += k.z < limit(i + 2);
      before += k.w < limit(i + 3);
    }
  };
  // (a row equal to mine counts where its token is in front: the same answer for all of a share but those around t)
  if (hi <= t0) count([&](int) { return mine + 1; });
  else if (lo >= t0 + tokens) count([&](int) { return mine; });
  else count([&](int i) { return mine + (i < t ? 1u : 0u); });
  counts[threadIdx.x] = before;
  __syncthreads();
  if (part == 0 && t < n) {
    uint32_t to = 0;
    for (int p = 0; p < parts; ++p) to += counts[p * tokens + at];
    keys[to] = mine;
    places[to] = (uint32_t)t;
  }
}

// A radix pass over digits of at most kDigitBits bits in three launches: every tile's counts of digits; for every digit
// their sums over the tiles in front; every tile's tokens to their places.  No atomics beyond a workgroup's counts, so
// the order is the same on every run.
constexpr int kSortThreads = 256, kSortEach = 4, kSortTile = kSortThreads * kSortEach;
constexpr int kDigitBits = 9, kDigits = 1 << kDigitBits;
constexpr int kSortWaves = kSortThreads / 64;

// Where a pass reads its rows and tokens: from the ids, or from what the pass before wrote.
struct EmbSource {
  EmbIds ids;
  const uint32_t* keys;
  const uint32_t* places;
  __device__ __forceinline__ uint32_t key(int64_t i) const { return keys ? keys[i] : ids.key(i); }
  __device__ __forceinline__ uint32_t place(int64_t i) const { return keys ? places[i] : (uint32_t)i; }
};

__global__ __launch_bounds__(kSortThreads) void embedding_count_kernel(EmbSource from, int64_t n, int shift, uint32_t* __restrict__ counts,
                                                                       uint32_t* __restrict__ chains, EmbRide ride) {
  if (rode<kSortThreads>(ride)) return;
  __shared__ uint32_t digits[kDigits];
  if (blockIdx.x == 0 && threadIdx.x == 0) *chains = 0;
  for (int d = threadIdx.x; d < kDigits; d += kSortThreads) digits[d] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * kSortTile;
#pragma unroll
  for (int k = 0; k < kSortEach; ++k) {
    const int64_t i = base + k * kSortThreads + threadIdx.x;
    if (i < n) atomicAdd(&digits[from.key(i) >> shift & (kDigits - 1)], 1u);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < kDigits; d += kSortThreads) counts[(int64_t)d * ride.own + blockIdx.x] = digits[d];
}

__device__ __forceinline__ uint32_t wave_running_sum(uint32_t v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t u = __shfl_up(v, off, 64);
    if (lane >= off) v += u;
  }
  return v;
}

// One wave a digit.
__global__ __launch_bounds__(kSortThreads) void embedding_offsets_kernel(uint32_t* __restrict__ counts, int64_t tiles,
                                                                         uint32_t* __restrict__ totals, EmbRide ride) {
  if (rode<kSortThreads>(ride)) return;
  const int lane = threadIdx.x & 63;
  const int64_t digit = (int64_t)blockIdx.x * kSortWaves + (threadIdx.x >> 6);
  uint32_t* mine = counts + digit * tiles;
  uint32_t sum = 0;
  for (int64_t base = 0; base < tiles; base += 64) {
    const int64_t i = base + lane;
    const uint32_t v = i < tiles ? mine[i] : 0u, upto = wave_running_sum(v);
    if (i < tiles) mine[i] = sum + upto - v;
    sum += __shfl(upto, 63, 64);
  }
  if (lane == 0) totals[digit] = sum;
}

__global__ __launch_bounds__(kSortThreads) void embedding_scatter_kernel(EmbSource from, int64_t n, int shift,
                                                                         const uint32_t* __restrict__ offsets,
                                                                         const uint32_t* __restrict__ totals,
                                                                         uint32_t* __restrict__ keys,
                                                                         uint32_t* __restrict__ places, EmbRide ride) {
  if (rode<kSortThreads>(ride)) return;
  __shared__ uint32_t counts[kSortWaves][kDigits];  // of a digit in a wave's tokens so far; then where the wave's begin
  __shared__ uint32_t sums[kSortWaves];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int d = threadIdx.x; d < kSortWaves * kDigits; d += kSortThreads) (&counts[0][0])[d] = 0;
  __syncthreads();
  uint32_t key[kSortEach], place[kSortEach], rank[kSortEach];
  const int64_t base = (int64_t)blockIdx.x * kSortTile + wave * 64 * kSortEach;  // (a wave's tokens lie side by side)
#pragma unroll
  for (int k = 0; k < kSortEach; ++k) {
    const int64_t i = base + k * 64 + lane;
    const bool in = i < n;
    key[k] = in ? from.key(i) : 0u;
    place[k] = in ? from.place(i) : 0u;
  }
#pragma unroll
  for (int k = 0; k < kSortEach; ++k) {
    const bool in = base + k * 64 + lane < n;
    const uint32_t d = key[k] >> shift & (kDigits - 1);
    uint64_t same = __ballot(in);  // the wave's lanes with this lane's digit
#pragma unroll
    for (int b = 0; b < kDigitBits; ++b) {
      const uint64_t ones = __ballot(d >> b & 1);
      same &= d >> b & 1 ? ones : ~ones;
    }
    const uint64_t front = same & ((1ull << lane) - 1);
    rank[k] = counts[wave][d] + (uint32_t)__popcll(front);
    __syncthreads();
    if (in && front == 0) counts[wave][d] += (uint32_t)__popcll(same);
    __syncthreads();
  }
  // where every digit's tokens of this tile begin: behind all smaller digits, and this digit's of the tiles in front
  constexpr int kEach = kDigits / kSortThreads;
  uint32_t total[kEach], sum = 0;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    total[e] = totals[threadIdx.x * kEach + e];
    sum += total[e];
  }
  const uint32_t upto = wave_running_sum(sum);
  if (lane == 63) sums[wave] = upto;
  __syncthreads();
  uint32_t at = upto - sum;
  for (int w = 0; w < wave; ++w) at += sums[w];
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int d = threadIdx.x * kEach + e;
    uint32_t here = at + offsets[(int64_t)d * ride.own + blockIdx.x];
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
      const uint32_t c = counts[w][d];
      counts[w][d] = here;
      here += c;
    }
    at += total[e];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kSortEach; ++k) {
    if (base + k * 64 + lane >= n) break;
    const uint32_t to = counts[wave][key[k] >> shift & (kDigits - 1)] + rank[k];
    keys[to] = key[k];
    places[to] = place[k];
  }
}

// ---- sums of equal rows.  A run of equal rows in the sorted tokens is cut into pieces of `chunk` tokens from its first
// token on, so that a row's sum depends on its own tokens alone, wherever its run lies.  A run of one piece is summed in
// order; the others are chains: their pieces but the first leave float32 sums in `parts`, and another launch joins them.
// The sorted tokens are cut into chunks of as many tokens; a workgroup sums the pieces that begin in its chunk (one at
// most of a run that began before, whose slot of `parts` is the chunk's).
struct EmbSums {
  const uint32_t* keys;
  const uint32_t* places;
  int64_t n, rows, cols, ldd;
  int chunk;        // tokens
  float scale;
  bool past;        // (see EmbRide)
  float* parts;     // [chunks][cols]
  uint32_t* chains; // how many; then the places that they begin at
};

constexpr int kChunkMost = 32;

// First place whose row is not below `key` (between lo and hi), by the whole wave: 64 probes a step.
__device__ __forceinline__ int64_t wave_lower_bound(const uint32_t* __restrict__ keys, int64_t lo, int64_t hi, uint32_t key) {
  const int lane = threadIdx.x & 63;
  while (lo < hi) {  // the answer is in [lo, hi]
    const int64_t step = (hi - lo + 63) / 64, at = lo + lane * step;
    const uint64_t below = __ballot(at < hi && keys[at < hi ? at : lo] < key);  // a prefix of the lanes
    const int many = __popcll(below);
    if (many == 0) return lo;
    const int64_t last = lo + (many - 1) * step;  // below the key
    hi = last + step < hi ? last + step : hi;
    lo = last + 1;
  }
  return lo;
}

template <class G>
__device__ __forceinline__ void store_row(G* to, int64_t left, const float* acc, float scale, bool past) {
  float f[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = acc[e] * scale;
  const Piece<G, 8> q = from_floats<G>(f);
  if (past) store_piece<true>(to, left, q);
  else store_piece<false>(to, left, q);
}

// A lane holds 8 columns, blockIdx.y says which of several slabs of blockDim.x * 8 columns; 8 tokens' pieces are asked for before the first is added.
template <class D, class G>
__global__ __launch_bounds__(256) void embedding_sums_kernel(EmbSums a, const D* __restrict__ dout, G* __restrict__ grad) {
  constexpr int V = 8, U = 8;
  __shared__ uint32_t keys[3 * kChunkMost + 2], places[2 * kChunkMost];
  const int64_t c = ((int64_t)blockIdx.y * blockDim.x + threadIdx.x) * V, left = a.cols - c;
  // The rows of the chunk's tokens, of `chunk` and one tokens in front of them and of `chunk` behind.
  const int C = a.chunk, lane = threadIdx.x & 63;
  const int64_t c0 = (int64_t)blockIdx.x * C;
  const int own = (int)(a.n - c0 < C ? a.n - c0 : C);
  const uint32_t none = (uint32_t)a.rows;  // tokens without a row lie behind all others
  for (int i = threadIdx.x; i < 3 * C + 2; i += blockDim.x) {
    const int64_t at = c0 - C - 1 + i;
    keys[i] = at >= 0 && at < a.n ? a.keys[at] : 0xFFFFFFFFu;
    if (i > C && i <= 3 * C) places[i - C - 1] = at < a.n ? a.places[at] : 0u;
  }
  __syncthreads();
  auto key = [&](int i) { return keys[i + C + 1]; };  // -C - 1 <= i <= 2 C
  // Every wave for itself, a lane a token: the first tokens of runs, and the first place of the piece [lead, ...) of
  // the run that began in front of the chunk, if one begins here.
  const uint64_t starts = __ballot(lane < own && key(lane < C ? lane : 0) != key(lane < C ? lane - 1 : 0));
  const uint32_t k0 = key(0);
  int lead = -1;
  if (!(starts & 1)) {
    if (k0 == none) return;
    int at;
    if (key(-C) != k0) {  // it began less than a piece ago
      at = C - __builtin_ctzll(~__ballot(lane < C && key(lane < C ? -1 - lane : 0) == k0));
    } else {
      const int64_t begin = wave_lower_bound(a.keys, 0, c0 - C, k0);
      at = (int)((C - (c0 - begin) % C) % C);
    }
    if (at < own && key(at) == k0) lead = at;
  }
  if (lead < 0 && !starts) return;
  const int lo = lead >= 0 ? lead : __builtin_ctzll(starts);
  // the last piece that begins here, and its end
  const int tail = starts ? 63 - __builtin_clzll(starts) : lead;
  const uint32_t kt = key(tail);
  const bool whole = key(tail + C) == kt;  // and the run goes on
  int hi = tail;
  if (starts && kt != none && whole) {
    if (threadIdx.x == 0 && blockIdx.y == 0) a.chains[1 + atomicAdd(a.chains, 1u)] = (uint32_t)(c0 + tail);
  } else if (kt != none) {
    hi = whole ? tail + C : tail + 1 + __builtin_ctzll(__ballot(lane < C && key(tail + 1 + (lane < C ? lane : 0)) != kt));
  }
  float acc[V] = {};
  for (int i0 = lo; i0 < hi; i0 += U) {
    Piece<D, V> p[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u < hi ? i0 + u : hi - 1;
      load_piece<true>(dout + (int64_t)places[i] * a.ldd + c, left, p[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u;
      if (i >= hi) break;
      const uint32_t k = key(i);
      float f[V];
      to_floats(p[u], f);
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] += f[e];
      if (i + 1 == hi || key(i + 1) != k) {
        if (lead >= 0 && k == k0) store_row(a.parts + (int64_t)blockIdx.x * a.cols + c, left, acc, 1.f, false);
        else store_row(grad + (int64_t)k * a.cols + c, left, acc, a.scale, a.past);
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] = 0.f;
      }
    }
  }
}

// The chains: the tokens of their first piece and the sums of the others, dealt out in turn to 8 groups of 32 lanes of 8
// columns each, whose sums are added in order.
constexpr int kChainGroups = 2048;

template <class D, class G>
__global__ __launch_bounds__(256) void embedding_chains_kernel(EmbSums a, const D* __restrict__ dout, G* __restrict__ grad) {
  constexpr int V = 8, kLanes = 32, kGroups = 256 / kLanes, kCols = kLanes * V;
  __shared__ float sums[kGroups][kCols];
  const int64_t slabs = (a.cols + kCols - 1) / kCols, items = (int64_t)a.chains[0] * slabs;
  const int group = threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t begin = a.chains[1 + item / slabs], slab = item % slabs;
    const int64_t c = slab * kCols + lane * V, left = a.cols - c;
    const uint32_t k = a.keys[begin];
    float acc[V] = {};
#pragma unroll 4
    for (int64_t i = group; i < a.chunk; i += kGroups) {
      Piece<D, V> p;
      load_piece<false>(dout + (int64_t)a.places[begin + i] * a.ldd + c, left, p);
      float f[V];
      to_floats(p, f);
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] += f[e];
    }
    const int64_t end = wave_lower_bound(a.keys, begin + a.chunk, a.n, k + 1);
    const int64_t pieces = (end - begin - 1) / a.chunk;  // behind the first
    const float* parts = a.parts + (begin / a.chunk + 1) * a.cols + c;
#pragma unroll 4
    for (int64_t i = group; i < pieces; i += kGroups) {
      Piece<float, V> p;
      load_piece<false>(parts + i * a.cols, left, p);
      float f[V];
      to_floats(p, f);
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] += f[e];
    }
#pragma unroll
    for (int e = 0; e < V; ++e) sums[group][lane * V + e] = acc[e];
    __syncthreads();
    if (group == 0) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        acc[e] = 0.f;
        for (int g = 0; g < kGroups; ++g) acc[e] += sums[g][lane * V + e];
      }
      store_row(grad + (int64_t)k * a.cols + c, left, acc, a.scale, false);
    }
    __syncthreads();
  }
}

// Tokens of a chunk: 32 (147456 tokens: sums 147 us and chains 23; 64: 155 and 21; 16: 141 and 38), fewer where there would
// not be a thousand chunks (8192 tokens: 8, sums 10 us, with 16 15).
static int emb_chunk(int64_t n) {
  int c = 8;
  while (c < kChunkMost && c * 1024 < n) c *= 2;
  return c;
}

// The workspace, in 256-byte pieces.
struct EmbPlan {
  int64_t tiles, chunks, parts;
  int passes, chunk;
  int64_t keys[2], places[2], counts, totals, used, chains, sums, bytes;
};
static EmbPlan emb_plan(int64_t n, int64_t rows, int64_t cols) {
  EmbPlan p{};
  if (n <= 0 || rows <= 0 || cols <= 0) return p;
  p.chunk = emb_chunk(n);
  p.chunks = (n + p.chunk - 1) / p.chunk;
  if (n > kRankMost) {
    int bits = 1;
    while (rows >> bits) ++bits;
    p.passes = (bits + kDigitBits - 1) / kDigitBits;
    p.tiles = (n + kSortTile - 1) / kSortTile;
  }
  auto take = [&](int64_t bytes) {
    const int64_t at = p.bytes;
    p.bytes += (bytes + 255) & ~int64_t{255};
    return at;
  };
  for (int k = 0; k < (p.passes > 1 ? 2 : 1); ++k) {
    p.keys[k] = take(4 * n);
    p.places[k] = take(4 * n);
  }
  if (p.passes) {
    p.counts = take(4 * kDigits * p.tiles);
    p.totals = take(4 * kDigits);
    p.used = take(rows);
  }
  p.chains = take(4 * (1 + p.chunks));
  p.sums = take(4 * p.chunks * cols);
  return p;
}

// Results that do not stay in the last cache (256 MB) until someone reads them are stored past it.
static bool emb_past(int64_t bytes) { return bytes > (int64_t{384} << 20); }

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
  const int64_t slabs = (cols + kEmbSlab - 1) / kEmbSlab;
  const int64_t groups = slabs > kEmbGroups * kEmbWaves / n ? kEmbGroups + 1 : (n * slabs + kEmbWaves - 1) / kEmbWaves;
  if (rows >= 0x7FFFFFFF || groups > kEmbGroups) return MX_ERR_UNSUPPORTED;
  const EmbIds e{ids, ids_i64 != 0, first, rows, 0};
  of_type(weight_f32, [&](auto w) {
    of_type(out_f32, [&](auto o) {
      if (cols <= 512) {
        const int shift = cols <= 64 ? 3 : cols <= 128 ? 4 : cols <= 256 ? 5 : 6;
        const int64_t per = (int64_t)(kEmbThreads >> shift) * kEmbTokens;
        hipLaunchKernelGGL((embedding_narrow_kernel<decltype(w), decltype(o)>), dim3((unsigned)((n + per - 1) / per)), dim3(kEmbThreads), 0,
                           (hipStream_t)stream, e, n, (const decltype(w)*)weight, cols, ldw, scale,
                           emb_past(n * cols * (out_f32 ? 4 : 2)), shift, (decltype(o)*)out);
        return;
      }
      hipLaunchKernelGGL((embedding_kernel<decltype(w), decltype(o)>), dim3((unsigned)groups), dim3(kEmbThreads), 0,
                         (hipStream_t)stream, e, n, (const decltype(w)*)weight, cols, ldw, scale,
                         emb_past(n * cols * (out_f32 ? 4 : 2)), (uint32_t)slabs, (decltype(o)*)out);
    });
  });
  return hipGetLastError() == hipSuccess ? MX_OK : MX_ERR_LAUNCH;
}

extern "C" int64_t mx_embedding_grad_workspace(int64_t n, int64_t rows, int64_t cols) {
  return emb_plan(n, rows, cols).bytes;
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
  const EmbPlan p = emb_plan(n, rows, cols);
  const int threads = cols > 1024 ? 256 : cols > 512 ? 128 : 64;
  const int64_t slabs = (cols + threads * 8 - 1) / (threads * 8), bytes = rows * cols * (grad_f32 ? 4 : 2);
  const int64_t row_bytes = cols * (grad_f32 ? 4 : 2), pieces = rows * ((row_bytes + 15) / 16);
  if (slabs > 65535 || ride_groups(pieces, 256) + p.tiles + kDigits > kEmbGroups || p.chunks > kEmbGroups || row_bytes > 0x7FFFFFFF)
    return MX_ERR_UNSUPPORTED;
  hipStream_t st = (hipStream_t)stream;
  uint8_t* ws = (uint8_t*)workspace;
  auto words = [&](int64_t at) { return (uint32_t*)(ws + at); };
  uint32_t* chains = words(p.chains);
  const EmbIds e{ids, ids_i64 != 0, first, rows, padding};
  const bool past = emb_past(bytes);
  uint8_t* out = (uint8_t*)grad;
  auto nothing = [&](unsigned own) { return EmbRide{kRideFill, own, out, 0, past, e, nullptr, 0, 0}; };
  auto fill = [&](unsigned own, uint8_t* to, int64_t from, int64_t many) {
    return EmbRide{kRideFill, own, to + from, many, past, e, nullptr, 0, 0};
  };
  auto launch = [&](const EmbRide& q, int lanes, auto&& f) {
    const int64_t riding = q.mode == kRideFill ? (q.count + 15) / 16 : q.count;
    f(dim3((unsigned)(q.own + ride_groups(riding, lanes))), dim3(lanes));
  };
  auto zeros = [&](int64_t from) {
    const EmbRide q = fill(0, out, from, bytes - from);
    if (q.count > 0)
      launch(q, 256, [&](dim3 g, dim3 b) { hipLaunchKernelGGL(embedding_zeros_kernel, g, b, 0, st, q); });
  };
  int last = 0;  // which of the two lists holds the order
  if (n == 0) {
    zeros(0);
    return hipGetLastError() == hipSuccess ? MX_OK : MX_ERR_LAUNCH;
  }
  if (p.passes == 0) {
    // Past the caches the launch's large workgroups fill at 5 TB/s: no more of the zeros there than the placing hides
    // (2003 tokens, 622 MB: 8 us less than with all of them; 8192 tokens, 311 MB through the caches: 5 more, so all).
    const int tokens = rank_tokens(n);
    const int64_t here = past ? std::min<int64_t>(bytes, int64_t{48} << 20) : bytes;
    const EmbRide q = fill((unsigned)((n + tokens - 1) / tokens), out, 0, here);
    launch(q, kRankThreads, [&](dim3 g, dim3 b) {
      hipLaunchKernelGGL(embedding_rank_kernel, g, b, 0, st, e, (int)n, tokens, words(p.keys[0]), words(p.places[0]), chains, q);
    });
    zeros(here);
  }
  // One pass: a small table, filled by the first launch.  More: the first launch clears the rows' flags, the second sets
  // them, the others share the unused rows' zeros.
  int launched = 0;
  const int64_t parts = 3 * p.passes - 2, share = parts > 0 ? (pieces + parts - 1) / parts : 0;
  auto ride = [&](unsigned own) {
    const int k = launched++;
    if (p.passes == 1) return k == 0 ? fill(own, out, 0, bytes) : nothing(own);
    if (k == 0) return fill(own, ws + p.used, 0, (rows + 255) & ~int64_t{255});
    if (k == 1) return EmbRide{kRideMark, own, ws + p.used, n, false, e, nullptr, 0, 0};
    const int64_t from = std::min(pieces, share * (k - 2));
    return EmbRide{kRideUnused, own, out, std::min(share, pieces - from), past, e, ws + p.used, from, row_bytes};
  };
  for (int pass = 0; pass < p.passes; ++pass) {
    EmbSource from{e, nullptr, nullptr};
    if (pass > 0) {
      from.keys = words(p.keys[last]);
      from.places = words(p.places[last]);
      last ^= 1;
    }
    const int shift = pass * kDigitBits;
    const EmbRide q0 = ride((unsigned)p.tiles), q1 = ride(kDigits / kSortWaves), q2 = ride((unsigned)p.tiles);
    launch(q0, kSortThreads, [&](dim3 g, dim3 b) {
      hipLaunchKernelGGL(embedding_count_kernel, g, b, 0, st, from, n, shift, words(p.counts), chains, q0);
    });
    launch(q1, kSortThreads, [&](dim3 g, dim3 b) {
      hipLaunchKernelGGL(embedding_offsets_kernel, g, b, 0, st, words(p.counts), p.tiles, words(p.totals), q1);
    });
    launch(q2, kSortThreads, [&](dim3 g, dim3 b) {
      hipLaunchKernelGGL(embedding_scatter_kernel, g, b, 0, st, from, n, shift, words(p.counts), words(p.totals),
                         words(p.keys[last]), words(p.places[last]), q2);
    });
  }
  const EmbSums a{words(p.keys[last]), words(p.places[last]), n, rows, cols, ldd, p.chunk, scale, past, (float*)(ws + p.sums),
                  chains};
  of_type(dout_f32, [&](auto dt) {
    of_type(grad_f32, [&](auto gt) {
      using D = decltype(dt);
      using G = decltype(gt);
      hipLaunchKernelGGL((embedding_sums_kernel<D, G>), dim3((unsigned)p.chunks, (unsigned)slabs), dim3(threads), 0, st, a,
                         (const D*)dout, (G*)grad);
      if (n > p.chunk)  // (a chain is more than one piece)
        hipLaunchKernelGGL((embedding_chains_kernel<D, G>), dim3(kChainGroups), dim3(256), 0, st, a, (const D*)dout, (G*)grad);
    });
  });
  return hipGetLastError() == hipSuccess ? MX_OK : MX_ERR_LAUNCH;
}
