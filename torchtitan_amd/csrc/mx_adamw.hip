// The AdamW step over a list of parameters, with moments in float32 or in 8 bits.
//
//   g = f * gradient,  f = min(1, limit / (N + 1e-6))           (f = 1 without a norm N)
//   m = b1 m + (1 - b1) g          v = b2 v + (1 - b2) g^2
//   w = (1 - lr decay) w - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Bound by memory: everything is read once and written once, 28 bytes a float32 parameter, 22 a bf16 one, 28 with a float32
// master weight beside it (2 more with float32 gradients of bf16 parameters).  In 8 bits the moments' 16 of these are 4.1.  A table
// of tensors travels as a kernel argument; a tensor is cut into chunks of one workgroup each.
//
// Moments in 8 bits: blocks of 32 in the order of memory, a power of two for each (a byte b: 2^(b - 127), 255: the block is
// NaN), chosen as the smallest with which the block's largest value is no more than the largest code.
//   m  e4m3 with a sign, bias 7, up to 448
//   v  e5m3 without one, bias 15, up to 122880 (of v itself: its root then has a code for every 2^17 below the block's
//      largest, as m has, so that m does not outlive v; a v that is not 0 keeps at least the smallest code)
// A value between two codes becomes the upper one with the probability of its distance from the lower.  Rounding to nearest
// would hold v still: a step changes it by (1 - b2) of itself, two orders below half a code; the two recursions are linear, so
// with this rounding the expected moments are those of float32.  The 16 random bits are a hash of the value's place, the
// parameter's number, the step and a seed: a run that is repeated or resumed gives the same bits.
#include <algorithm>
#include <cmath>
#include <utility>
#include <vector>

#include "mx_rows.h"

namespace mx {

constexpr int kAdamThreads = 256;
constexpr int kAdamTensors = 44;  // of one launch
// Pieces a lane and chunk of parameters with moments in float32: 4, or 1 where the list has no more than 2^20 values, a chunk of 4 for
// every CU (271 000 values 8.5 us with 4, 4.5 with 1; 673 million 3.39 ms with 4, 3.51 with 1).
constexpr int kAdamPieces = 4;
constexpr int64_t kAdamFew = 1 << 20;
constexpr int kAdamValues = 4;  // values a piece: 16 bytes of float32
// With moments in 8 bits, values a lane and chunk: 16, or 8 for such lists (us in a graph with 8 and 16, float32: 65 536 values 3.7 and 4.5,
// 271 000 3.9 and 4.9, 2^20 4.9 and 5.2, 2^21 7.3 and 7.5, 2^22 11.8 and 12.4; bf16 3.6 and 4.3, 3.9 and 4.8, 4.7 and 4.7, 6.3 and 6.9,
// 10 and 10.4; 50 million 94 and 95, 673 million 1265 and 1198, float32 2102 and 2051).
constexpr int kAdam8Few = 8, kAdam8Values = 16;

struct AdamEntry {
  void* p;
  const void* g;
  void *m, *v;         // float32, or codes
  uint8_t *ms, *vs;    // scales of codes
  float* master;       // or null
  int64_t elems;
  uint32_t first;      // first chunk of this tensor
  uint32_t key;        // of its random bits; its number where the corrections are on the device
  float step, root;    // lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
  uint32_t types;      // of parameter and gradient: 0 bf16, 1 float32, 2 bf16 and float32
};
struct AdamTable {
  AdamEntry e[kAdamTensors];
};
struct AdamHyper {
  float b1, c1, b2, c2, eps, decay;  // c: 1 - b; decay: 1 - lr * weight decay
  float sign, limit;
  const float* norm;           // or null
  const float4* corrections;   // or null: step, root, decay, key of every number
};

__host__ __device__ __forceinline__ uint32_t adam_mix(uint32_t x) {
  x = (x ^ (x >> 16)) * 0x6A09E667u;
  x = (x ^ (x >> 15)) * 0xBB67AE85u;
  return x ^ (x >> 16);
}
__host__ __device__ __forceinline__ uint32_t adam_key(uint64_t seed, uint32_t step, uint32_t number) {
  uint32_t key = 0;
  for (const uint32_t word : {(uint32_t)seed, (uint32_t)(seed >> 32), step, number}) key = adam_mix(key + word + 0x9E3779B9u);
  return key;
}

__device__ __forceinline__ int adam_find(const AdamTable& t, int n, uint32_t chunk) {
  int lo = 0, hi = n;  // the last entry whose first chunk is not behind this one
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.e[mid].first <= chunk) lo = mid; else hi = mid;
  }
  return lo;
}

// V values at p, from any element on; ALL: they exist, else `left` of them do (the others: 0).
template <bool ALL, int V, class T>
__device__ __forceinline__ void adam_load(const T* p, int64_t left, float (&f)[V]) {
  constexpr int W = V * (int)sizeof(T) / 4;
  typedef uint32_t words __attribute__((ext_vector_type(W > 4 ? 4 : W), aligned(sizeof(T))));
  if (ALL || left >= V) {
    uint32_t w[W];
#pragma unroll
    for (int k = 0; k < W; k += 4) {
      const words q = __builtin_nontemporal_load(reinterpret_cast<const words*>(p) + k / 4);
#pragma unroll
      for (int j = 0; j < (W > 4 ? 4 : W); ++j) w[k + j] = q[j];
    }
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if constexpr (sizeof(T) == 4) f[e] = __uint_as_float(w[e]);
      else f[e] = e & 1 ? bf16_hi(w[e / 2]) : bf16_lo(w[e / 2]);
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < V; ++e) {
    f[e] = 0.f;
    if (e < left) {
      if constexpr (sizeof(T) == 4) f[e] = p[e];
      else f[e] = bf16_lo(p[e]);
    }
  }
}
template <bool ALL, int V, class T>
__device__ __forceinline__ void adam_store(T* p, int64_t left, const float (&f)[V]) {
  constexpr int W = V * (int)sizeof(T) / 4;
  typedef uint32_t words __attribute__((ext_vector_type(W > 4 ? 4 : W), aligned(sizeof(T))));
  uint32_t w[W];
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < V; ++e) w[e] = __float_as_uint(f[e]);
  } else {
#pragma unroll
    for (int e = 0; e < V; e += 2)
      w[e / 2] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f_t{f[e], f[e + 1]}, v2bf_t));
  }
  if (ALL || left >= V) {
#pragma unroll
    for (int k = 0; k < W; k += 4) {
      words q;
#pragma unroll
      for (int j = 0; j < (W > 4 ? 4 : W); ++j) q[j] = w[k + j];
      __builtin_nontemporal_store(q, reinterpret_cast<words*>(p) + k / 4);
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < V; ++e)
    if (e < left) {
      if constexpr (sizeof(T) == 4) p[e] = f[e];
      else p[e] = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
    }
}

// The new moments and weight of one value.  Products and sums are rounded one by one, as separate operations on tensors
// round them: the same bits as the formula in torch operations.
// ROUGH: the hardware's root and reciprocal, each within an ulp, for an eps (from 1e-9 on) that covers what they lose of a
// denormal second moment, and then for every value of the call, whichever chunk it is in; the sequences around them that round right
// took 7 to 15 % of the time of a bf16 parameter with moments in 8 bits (us with them and without: 673 million 1329 and 1251, 50 million
// 107 and 91), and nothing elsewhere.
template <bool ROUGH>
__device__ __forceinline__ void adam_update(const AdamHyper& h, float f, float step, float root, float decay, float g, float& m,
                                            float& v, float& w) {
#pragma clang fp contract(off)
  g = g * f;
  m = m * h.b1 + g * h.c1;
  v = v * h.b2 + g * g * h.c2;
  if constexpr (ROUGH) {
    const float below = __builtin_amdgcn_sqrtf(v) * root + h.eps;
    w = w * decay - step * (m * __builtin_amdgcn_rcpf(below));
  } else {
    const float below = __builtin_sqrtf(v) * root + h.eps;
    w = w * decay - step * (m / below);
  }
}

// T: the parameter's values, G: its gradient's
template <bool ALL, int PIECES, class T, class G>
__device__ __forceinline__ void adam_chunk(const AdamEntry& e, const AdamHyper& h, float f, float step, float root, float decay,
                                           int64_t at) {
  constexpr int V = kAdamValues;
  const G* g = (const G*)e.g;
  T* p = (T*)e.p;
  float *m = (float*)e.m, *v = (float*)e.v;
  float qg[PIECES][V], qm[PIECES][V], qv[PIECES][V], qw[PIECES][V];
  auto pieces = [&](auto&& piece) {
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
      const int64_t i = at + (k * kAdamThreads + threadIdx.x) * V;
      piece(k, i, e.elems - i);
    }
  };
  // one array after the other
  pieces([&](int k, int64_t i, int64_t left) { adam_load<ALL>(g + i, left, qg[k]); });
  pieces([&](int k, int64_t i, int64_t left) { adam_load<ALL>(m + i, left, qm[k]); });
  pieces([&](int k, int64_t i, int64_t left) { adam_load<ALL>(v + i, left, qv[k]); });
  if (e.master) pieces([&](int k, int64_t i, int64_t left) { adam_load<ALL>(e.master + i, left, qw[k]); });
  else pieces([&](int k, int64_t i, int64_t left) { adam_load<ALL>((const T*)p + i, left, qw[k]); });
#pragma unroll
  for (int k = 0; k < PIECES; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) adam_update<false>(h, f, step, root, decay, qg[k][j], qm[k][j], qv[k][j], qw[k][j]);
  pieces([&](int k, int64_t i, int64_t left) { adam_store<ALL>(m + i, left, qm[k]); });
  pieces([&](int k, int64_t i, int64_t left) { adam_store<ALL>(v + i, left, qv[k]); });
  if (e.master) pieces([&](int k, int64_t i, int64_t left) { adam_store<ALL>(e.master + i, left, qw[k]); });
  pieces([&](int k, int64_t i, int64_t left) { adam_store<ALL>(p + i, left, qw[k]); });
}

__device__ __forceinline__ float adam_factor(const AdamHyper& h) {
  if (!h.norm) return h.sign;
  const float f = (1.f / (*h.norm + 1e-6f)) * h.limit;  // (a reciprocal and a product, as torch divides a number by a tensor)
  return h.sign * (f > 1.f ? 1.f : f);  // (NaN stays)
}

// ---- 8 bits.  A code's bits are the topmost bits of a float32 whose exponent is the code's: a value times 2^(bias - b), b the
// block's scale byte, has its code in bits 20 and up (what lies below the smallest normal code is a denormal float32, whose
// bits go on in the same steps), so that rounding is an addition and a shift, and decoding a shift and a multiplication.
constexpr int kFirstBias = 7, kSecondBias = 15;      // of the codes' exponents
constexpr int kFirstTop = 8, kSecondTop = 16;        // exponent of the largest code
constexpr uint32_t kFirstMost = 0x7E, kSecondMost = 0xFF;
constexpr uint32_t kFirstUp = 0x1FFFFF, kSecondUp = 0x0FFFFF;  // carries a mantissa above the largest code's

__device__ __forceinline__ float adam_decode1(uint32_t code, int scale) {  // code 0 .. 255
  const float x = __builtin_amdgcn_ldexpf(__uint_as_float((code & 127u) << 20), scale - kFirstBias);
  return __uint_as_float(__float_as_uint(x) | (code >> 7) << 31);
}
__device__ __forceinline__ float adam_decode2(uint32_t code, int scale) {
  return __builtin_amdgcn_ldexpf(__uint_as_float(code << 20), scale - kSecondBias);
}
// The scale byte of a block whose largest magnitude has these bits.
__device__ __forceinline__ int adam_scale(uint32_t amax, uint32_t up, int top) {
  if (amax >= 0x7F800000u) return 255;
  const int b = (int)((amax + up) >> 23) - top;
  return amax == 0 || b < 0 ? 0 : b;  // (at most 255 - 8, which is below 255)
}
// Largest magnitude bits of a block: V values here, 32 / V lanes.
template <int V>
__device__ __forceinline__ uint32_t adam_block_max(const float (&x)[V]) {
  uint32_t a = 0;
#pragma unroll
  for (int j = 0; j < V; ++j) a = max(a, __float_as_uint(x[j]) & 0x7FFFFFFFu);
  a = max(a, dpp<kQuadXor1>(a));
  a = max(a, dpp<kQuadXor2>(a));
  return V == 8 ? a : max(a, dpp<kRowHalfMirror>(a));
}

// Four codes of a first moment as values of scale 1.
__device__ __forceinline__ void adam_decode_first(uint32_t codes, float* x) {
  const v2f_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
  x[0] = lo.x, x[1] = lo.y, x[2] = hi.x, x[3] = hi.y;
}

// V values a piece: 8 of a bf16 parameter, 4 of a float32 one, so that either is 16 bytes (float32, 8 / 4: 50 million 167 / 138 us,
// 673 million 2.06 / 2.12 ms).
template <bool ALL, bool ROUGH, int VALUES, int V, class T, class G>
__device__ __forceinline__ void adam8_chunk(const AdamEntry& e, const AdamHyper& h, float f, float step, float root, float decay,
                                            uint32_t key, int64_t at) {
  constexpr int kPieces = VALUES / V, kWords = V / 4;
  typedef uint32_t Codes __attribute__((ext_vector_type(kWords)));
  const G* g = (const G*)e.g;
  T* p = (T*)e.p;
  uint8_t *m = (uint8_t*)e.m, *v = (uint8_t*)e.v;
  const int64_t whole = (e.elems + 31) & ~int64_t{31};  // codes are whole blocks
  float qg[kPieces][V], qw[kPieces][V];
  Codes cm[kPieces], cv[kPieces];
  int sm[kPieces], sv[kPieces];
  auto pieces = [&](auto&& piece) {
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
      const int64_t i = at + (k * kAdamThreads + threadIdx.x) * V;
      piece(k, i, e.elems - i);
    }
  };
  auto codes = [&](Codes(&c)[kPieces], const uint8_t* from) {
    pieces([&](int k, int64_t i, int64_t) {
      c[k] = Codes(0);
      if (ALL || i < whole) c[k] = __builtin_nontemporal_load(reinterpret_cast<const Codes*>(from + i));
    });
  };
  auto scales = [&](int(&s)[kPieces], const uint8_t* from) {
    pieces([&](int k, int64_t i, int64_t) { s[k] = ALL || i < whole ? from[i >> 5] : 0; });
  };
  // one array after the other
  pieces([&](int k, int64_t i, int64_t left) { adam_load<ALL>(g + i, left, qg[k]); });
  if (e.master) pieces([&](int k, int64_t i, int64_t left) { adam_load<ALL>(e.master + i, left, qw[k]); });
  else pieces([&](int k, int64_t i, int64_t left) { adam_load<ALL>((const T*)p + i, left, qw[k]); });
  codes(cm, m);
  codes(cv, v);
  scales(sm, e.ms);
  scales(sv, e.vs);
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    const int64_t i = at + (k * kAdamThreads + threadIdx.x) * V, left = e.elems - i;
    float fm[V], fv[V];
#pragma unroll
    for (int j = 0; j < kWords; ++j) adam_decode_first(cm[k][j], fm + 4 * j);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      fm[j] = __builtin_amdgcn_ldexpf(fm[j], sm[k] - 127);
      fv[j] = adam_decode2(cv[k][j / 4] >> (8 * (j & 3)) & 255u, sv[k]);
    }
    if (sm[k] == 255 || sv[k] == 255) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (sm[k] == 255) fm[j] = __builtin_nanf("");
        if (sv[k] == 255) fv[j] = __builtin_nanf("");
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      adam_update<ROUGH>(h, f, step, root, decay, qg[k][j], fm[j], fv[j], qw[k][j]);
      if (!ALL && j >= left) fm[j] = fv[j] = 0.f;  // (values that the last block does not have)
    }
    if (e.master) adam_store<ALL>(e.master + i, left, qw[k]);
    adam_store<ALL>(p + i, left, qw[k]);
    const int s1 = adam_scale(adam_block_max(fm), kFirstUp, kFirstTop), s2 = adam_scale(adam_block_max(fv), kSecondUp, kSecondTop);
    Codes o1 = Codes(0), o2 = Codes(0);
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      const uint32_t random = adam_mix((uint32_t)((i + j) >> 1) * 0x9E3779B9u + key);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        // (0 stays 0: what is added is less than a code)
        const uint32_t up = (q ? random >> 16 << 4 : (random & 0xFFFFu) << 4) | 8u;
        const uint32_t x = __float_as_uint(fm[j + q]);
        const uint32_t a = __float_as_uint(__builtin_amdgcn_ldexpf(__builtin_fabsf(fm[j + q]), kFirstBias - s1)) + up;
        const uint32_t b = __float_as_uint(__builtin_amdgcn_ldexpf(fv[j + q], kSecondBias - s2)) + up;
        const uint32_t code1 = min(a >> 20, kFirstMost) | (x >> 31 << 7);
        const uint32_t code2 = min(max(b >> 20, min(__float_as_uint(fv[j + q]), 1u)), kSecondMost);
        o1[j / 4] |= code1 << (8 * ((j + q) & 3));
        o2[j / 4] |= code2 << (8 * ((j + q) & 3));
      }
    }
    if (s1 == 255) o1 = (o1 & 0x80808080u) | 0x7E7E7E7Eu;
    if (s2 == 255) o2 = Codes(0xFFFFFFFFu);
    if (ALL || i < whole) {
      __builtin_nontemporal_store(o1, reinterpret_cast<Codes*>(m + i));
      __builtin_nontemporal_store(o2, reinterpret_cast<Codes*>(v + i));
      if ((threadIdx.x & (32 / V - 1)) == 0) {
        e.ms[i >> 5] = (uint8_t)s1;
        e.vs[i >> 5] = (uint8_t)s2;
      }
    }
  }
}

// PIECES a lane and chunk; with moments in 8 bits values.
template <bool EIGHT, int PIECES>
__global__ __launch_bounds__(kAdamThreads) void adamw_kernel(AdamTable table, int n, AdamHyper h) {
  const uint32_t chunk = blockIdx.x;
  const AdamEntry& e = table.e[adam_find(table, n, chunk)];
  float step = e.step, root = e.root, decay = h.decay;
  uint32_t key = e.key;
  if (h.corrections) {
    const float4 c = h.corrections[key];
    step = c.x, root = c.y, decay = c.z, key = __float_as_uint(c.w);
  }
  const float f = adam_factor(h);
  constexpr int kValues = kAdamThreads * PIECES * (EIGHT ? 1 : kAdamValues);
  const int64_t at = (int64_t)(chunk - e.first) * kValues;
  const bool all = e.elems - at >= kValues;
  auto types = [&](auto whole) {
    constexpr bool ALL = decltype(whole)::value;
    if constexpr (EIGHT) {
      if (h.eps < 1e-9f) {
        if (e.types == 1) adam8_chunk<ALL, false, PIECES, 4, float, float>(e, h, f, step, root, decay, key, at);
        else if (e.types == 0) adam8_chunk<ALL, false, PIECES, 8, uint16_t, uint16_t>(e, h, f, step, root, decay, key, at);
        else adam8_chunk<ALL, false, PIECES, 8, uint16_t, float>(e, h, f, step, root, decay, key, at);
      } else {
        if (e.types == 1) adam8_chunk<ALL, true, PIECES, 4, float, float>(e, h, f, step, root, decay, key, at);
        else if (e.types == 0) adam8_chunk<ALL, true, PIECES, 8, uint16_t, uint16_t>(e, h, f, step, root, decay, key, at);
        else adam8_chunk<ALL, true, PIECES, 8, uint16_t, float>(e, h, f, step, root, decay, key, at);
      }
    } else {
      if (e.types == 1) adam_chunk<ALL, PIECES, float, float>(e, h, f, step, root, decay, at);
      else if (e.types == 0) adam_chunk<ALL, PIECES, uint16_t, uint16_t>(e, h, f, step, root, decay, at);
      else adam_chunk<ALL, PIECES, uint16_t, float>(e, h, f, step, root, decay, at);
    }
  };
  if (all) types(std::true_type());
  else types(std::false_type());
}

// Step counters on the device: one more, and what follows from it, for every tensor of the table.
__global__ __launch_bounds__(64) void adamw_corrections_kernel(AdamTable table, int n, float* __restrict__ steps, double lr_host,
                                                               const float* __restrict__ lr_device, double b1, double b2,
                                                               double weight_decay, uint64_t seed, float4* __restrict__ out) {
  const int i = threadIdx.x;
  if (i >= n) return;
  const uint32_t number = table.e[i].key;
  const float t = steps[number] + 1.f;
  steps[number] = t;
  const double lr = lr_device ? (double)*lr_device : lr_host;
  const double one = 1.0 - pow(b1, (double)t), two = 1.0 - pow(b2, (double)t);
  out[number] = {(float)(lr / one), (float)(1.0 / sqrt(two)), (float)(1.0 - lr * weight_decay),
                 __uint_as_float(adam_key(seed, (uint32_t)t, number))};
}

// ---- the values that 8-bit moments stand for
constexpr int kMomentTensors = 96;
struct MomentEntry {
  const uint8_t *codes, *scales;
  void* out;
  int64_t elems;
  uint32_t first, kind;  // bit 0: the second moment, bit 1: out is float32
};
struct MomentTable {
  MomentEntry e[kMomentTensors];
};
constexpr int kMomentChunk = kAdamThreads * 8 * 2;

__global__ __launch_bounds__(kAdamThreads) void adamw_moments_kernel(MomentTable table, int n) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (table.e[mid].first <= blockIdx.x) lo = mid; else hi = mid;
  }
  const MomentEntry& e = table.e[lo];
  const int64_t at = (int64_t)(blockIdx.x - e.first) * kMomentChunk;
  const int64_t whole = (e.elems + 31) & ~int64_t{31};
  u32x2 c[2];
  int s[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int64_t i = at + (k * kAdamThreads + threadIdx.x) * 8;
    c[k] = u32x2{0, 0};
    s[k] = 0;
    if (i < whole) {
      c[k] = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(e.codes + i));
      s[k] = e.scales[i >> 5];
    }
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int64_t i = at + (k * kAdamThreads + threadIdx.x) * 8, left = e.elems - i;
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t code = c[k][j / 4] >> (8 * (j & 3)) & 255u;
      x[j] = e.kind & 1 ? adam_decode2(code, s[k]) : adam_decode1(code, s[k]);
      if (s[k] == 255) x[j] = __builtin_nanf("");
    }
    if (e.kind & 2) adam_store<false>((float*)e.out + i, left, x);
    else adam_store<false>((uint16_t*)e.out + i, left, x);
  }
}

// Whether two of the parameters share memory (where that cannot be found out: yes, the slower answer).
static bool adam_overlap(int64_t n, const int64_t* table) try {
  std::vector<std::pair<uintptr_t, uintptr_t>> runs;
  runs.reserve(n);
  for (int64_t i = 0; i < n; ++i) {
    const int64_t* t = table + i * MX_ADAMW_FIELDS;
    if (t[8]) runs.emplace_back((uintptr_t)t[0], (uintptr_t)t[0] + t[8] * (t[1] == 1 ? 4 : 2));
  }
  std::sort(runs.begin(), runs.end());
  for (size_t i = 1; i < runs.size(); ++i)
    if (runs[i].first < runs[i - 1].second) return true;
  return false;
} catch (...) {
  return true;
}

}  // namespace mx

using namespace mx;

extern "C" int mx_adamw(int64_t n, const int64_t* table, int eight, double lr, double beta1, double beta2, double eps,
                        double weight_decay, int maximize, const float* norm, float limit, uint64_t seed, float* steps,
                        const float* lr_device, void* corrections, void* stream) {
  if (n < 0 || (n > 0 && !table) || !(beta1 >= 0 && beta1 < 1) || !(beta2 >= 0 && beta2 < 1)) return MX_ERR_INVALID_ARG;
  if (((uintptr_t)norm & 3) || ((uintptr_t)steps & 3) || ((uintptr_t)lr_device & 3) || ((uintptr_t)corrections & 15))
    return MX_ERR_ALIGNMENT;
  if ((steps != nullptr) != (corrections != nullptr) || (lr_device && !steps)) return MX_ERR_INVALID_ARG;
  int64_t values = 0;
  for (int64_t i = 0; i < n; ++i) {
    const int64_t* t = table + i * MX_ADAMW_FIELDS;
    const int64_t elems = t[8], number = t[10];
    if (t[1] < 0 || t[1] > 2 || elems < 0 || number < 0 || number > 0x7FFFFFFF || (!steps && t[9] < 1)) return MX_ERR_INVALID_ARG;
    if (elems == 0) continue;
    if (!t[0] || !t[2] || !t[3] || !t[4] || (eight && (!t[5] || !t[6]))) return MX_ERR_INVALID_ARG;
    if (t[0] & (t[1] == 1 ? 3 : 1) || t[2] & (t[1] ? 3 : 1) || (t[3] | t[4]) & (eight ? 7 : 3) || t[7] & 3) return MX_ERR_ALIGNMENT;
    // (a place is hashed in 32 bits, two values at a time)
    if (elems >= int64_t{1} << 33) return MX_ERR_UNSUPPORTED;
    values = values > kAdamFew ? values : values + elems;
  }
  const bool few = values <= kAdamFew;
  const int64_t per = kAdamThreads * (eight ? (few ? kAdam8Few : kAdam8Values) : (few ? 1 : kAdamPieces) * kAdamValues);
  hipStream_t st = (hipStream_t)stream;
  AdamHyper h = {(float)beta1, (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), (float)eps,
                 (float)(1.0 - lr * weight_decay), maximize ? -1.f : 1.f, limit, norm, (const float4*)corrections};
  // parameters that share memory are updated one after the other, as a loop over them would
  const int most = adam_overlap(n, table) ? 1 : kAdamTensors;
  AdamTable args;
  int used = 0;
  int64_t chunks = 0;
  auto flush = [&]() -> int {
    if (used == 0) return MX_OK;
    if (steps)
      hipLaunchKernelGGL(adamw_corrections_kernel, dim3(1), dim3(64), 0, st, args, used, steps, lr, lr_device, beta1, beta2,
                         weight_decay, seed, (float4*)corrections);
    if (chunks) {
      const dim3 grid((unsigned)chunks), block(kAdamThreads);
      if (eight && few) hipLaunchKernelGGL((adamw_kernel<true, kAdam8Few>), grid, block, 0, st, args, used, h);
      else if (eight) hipLaunchKernelGGL((adamw_kernel<true, kAdam8Values>), grid, block, 0, st, args, used, h);
      else if (few) hipLaunchKernelGGL((adamw_kernel<false, 1>), grid, block, 0, st, args, used, h);
      else hipLaunchKernelGGL((adamw_kernel<false, kAdamPieces>), grid, block, 0, st, args, used, h);
    }
    used = 0;
    chunks = 0;
    return hipGetLastError() == hipSuccess ? MX_OK : MX_ERR_LAUNCH;
  };
  for (int64_t i = 0; i < n; ++i) {
    const int64_t* t = table + i * MX_ADAMW_FIELDS;
    const int64_t elems = t[8], mine = (elems + per - 1) / per;
    if (elems == 0 && !steps) continue;
    // (a launch has fewer than 2^32 lanes; a tensor of 2^33 values alone has no more than 2^23 chunks)
    if (used == most || chunks + mine > 0xFFFFFF)
      if (const int rc = flush()) return rc;
    AdamEntry& e = args.e[used++];
    e = {(void*)t[0], (const void*)t[2], (void*)t[3], (void*)t[4], (uint8_t*)t[5], (uint8_t*)t[6], (float*)t[7], elems,
         (uint32_t)chunks, (uint32_t)t[10], 0.f, 0.f, (uint32_t)t[1]};
    if (!steps) {
      const double at = (double)t[9];
      e.step = (float)(lr / (1.0 - std::pow(beta1, at)));
      e.root = (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, at)));
      e.key = adam_key(seed, (uint32_t)t[9], (uint32_t)t[10]);
    }
    chunks += mine;
  }
  return flush();
}

extern "C" int mx_adamw_moments(int64_t n, const uint8_t* const* codes, const uint8_t* const* scales, const int64_t* elems,
                                const int32_t* kinds, void* const* out, void* stream) {
  if (n < 0 || (n > 0 && (!codes || !scales || !elems || !kinds || !out))) return MX_ERR_INVALID_ARG;
  for (int64_t i = 0; i < n; ++i) {
    if (elems[i] < 0 || kinds[i] < 0 || kinds[i] > 3 || (elems[i] > 0 && (!codes[i] || !scales[i] || !out[i])))
      return MX_ERR_INVALID_ARG;
    if (((uintptr_t)codes[i] & 7) || ((uintptr_t)out[i] & (kinds[i] & 2 ? 3 : 1))) return MX_ERR_ALIGNMENT;
    if (elems[i] >= int64_t{1} << 33) return MX_ERR_UNSUPPORTED;
  }
  MomentTable args;
  int used = 0;
  int64_t chunks = 0;
  auto flush = [&]() -> int {
    if (used == 0) return MX_OK;
    hipLaunchKernelGGL(adamw_moments_kernel, dim3((unsigned)chunks), dim3(kAdamThreads), 0, (hipStream_t)stream, args, used);
    used = 0;
    chunks = 0;
    return hipGetLastError() == hipSuccess ? MX_OK : MX_ERR_LAUNCH;
  };
  for (int64_t i = 0; i < n; ++i) {
    if (elems[i] == 0) continue;
    const int64_t mine = (elems[i] + kMomentChunk - 1) / kMomentChunk;
    if (used == kMomentTensors || chunks + mine > 0xFFFFFF)
      if (const int rc = flush()) return rc;
    args.e[used++] = {codes[i], scales[i], out[i], elems[i], (uint32_t)chunks, (uint32_t)kinds[i]};
    chunks += mine;
  }
  return flush();
}
