// Kernels of the training graph's normalisation and regularisation: group normalisation with an activation and dropout,
// channels last.  x [N, P, C] (P = H * W pixels with a pixel stride of xcs elements), G groups of D = C / G channels:
//
//   mean[n,g], rstd[n,g] = 1 / sqrt(var + eps) over the P * D values of a group (biased variance)
//   xh = (x - mean) * rstd,  z = xh * gamma[c] + beta[c],  y = drop(act(z))
//   backward: dz = drop(dy) * act'(z);  A[n,c] = sum_p dz,  B[n,c] = sum_p dz * xh;  dbeta = sum_n A,  dgamma = sum_n B
//             dx = rstd * (dz * gamma - S1 / (P D) - xh * S2 / (P D)),  S1[n,g] = sum_{c in g} gamma A,  S2 = sum gamma B
//
// Every sum, statistic and intermediate is float32 (the merges over workgroups float64); only y and dx are rounded, once, to the
// tensors' type.  There are no atomics: partial results go through the workspace and are joined in a fixed order, so a call's
// results are the same bits every time.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fisr {

typedef _Float16 f16_t;
typedef __bf16 b16_t;
enum { NORM_ACT_NONE = 0, NORM_ACT_RELU = 1, NORM_ACT_SILU = 2, NORM_ACT_GELU = 3 };

// ---- the generator: Philox4x32 with 7 rounds (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011) ----
// 7 rounds are the fewest that the paper reports to pass all of BigCrush.  Block b of call `offset` under key `seed` is four words =
// eight 16-bit numbers; element i of a dense tensor has number i & 7 of block i >> 3 (word (i & 7) >> 1, low half first) and is dropped
// where it is below thresh = round(65536 p).  16 bits an element: a block costs 14 quarter-rate multiplies, which at 32 bits an
// element would take longer than a 16-bit tensor takes to stream; the rate that is realised, thresh / 65536, is what the scale of the
// kept values, 65536 / (65536 - thresh), goes by.
struct DropArgs {
  uint32_t thresh;                   // 0: no dropout
  float scale;
  uint64_t seed, offset;
  const uint64_t* counter;           // nullable, device: its value is added to offset when the kernel runs (captured graphs)
};
struct Philox { uint32_t w[4]; };
__device__ __forceinline__ Philox philox7(uint64_t block, uint64_t offset, uint64_t seed) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    const uint64_t p0 = (uint64_t)0xD2511F53u * c0, p1 = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)p1;
    c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return Philox{{c0, c1, c2, c3}};
}
__device__ __forceinline__ uint32_t philox_number(const Philox& r, int e) { return (e & 1) ? r.w[e >> 1] >> 16 : r.w[e >> 1] & 0xffffu; }

// v[e] is element i + e of the dense tensor: scaled where it is kept, zero (whatever it was: NaN and infinities too) where not.
// i % V == 0 and V divides 8, so the V elements share a block.
template <int V> __device__ __forceinline__ void drop_apply(float (&v)[V], uint64_t i, const DropArgs& d, uint64_t offset) {
  const Philox r = philox7(i >> 3, offset, d.seed);
  if (V == 8) {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = philox_number(r, e) >= d.thresh ? v[e] * d.scale : 0.f;
  } else {
    const int at = (int)(i & 7);
    const uint32_t lo = at & 4 ? r.w[2] : r.w[0], hi = at & 4 ? r.w[3] : r.w[1];      // (selects: an index would go through scratch)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int k = (at & 3) + e;                                                         // 0..3 within the pair of words
      const uint32_t w = k & 2 ? hi : lo, number = k & 1 ? w >> 16 : w & 0xffffu;
      v[e] = number >= d.thresh ? v[e] * d.scale : 0.f;
    }
  }
}

// ---- loads and stores of V channels as floats.  The caller sees to alignment: 16 bytes, or V elements where that is less ----
template <typename T, int V> struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) Pack { T e[V]; };
template <typename T, int V> __device__ __forceinline__ void load_v(const T* p, float (&v)[V]) {
  const Pack<T, V> q = *reinterpret_cast<const Pack<T, V>*>(p);
#pragma unroll
  for (int e = 0; e < V; ++e) v[e] = (float)q.e[e];
}
template <typename T, int V> __device__ __forceinline__ void store_v(T* p, const float (&v)[V]) {
  Pack<T, V> q;
#pragma unroll
  for (int e = 0; e < V; ++e) q.e[e] = (T)v[e];
  *reinterpret_cast<Pack<T, V>*>(p) = q;
}

template <typename T, int V> __device__ __forceinline__ void widen(const Pack<T, V>& q, float (&v)[V]) {
#pragma unroll
  for (int e = 0; e < V; ++e) v[e] = (float)q.e[e];
}
// Streaming forms (non-temporal): what is read or written once and is larger than the caches hold.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <typename T, int V> __device__ __forceinline__ Pack<T, V> load_nt(const T* p) {
  constexpr int B = sizeof(T) * V;
  Pack<T, V> q;
  if constexpr (B >= 16) {
    struct Q { u32x4 w[B / 16]; } u;
#pragma unroll
    for (int k = 0; k < B / 16; ++k) u.w[k] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p) + k);
    q = __builtin_bit_cast(Pack<T, V>, u);
  } else if constexpr (B == 8) {
    q = __builtin_bit_cast(Pack<T, V>, __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(p)));
  } else if constexpr (B == 4) {
    q = __builtin_bit_cast(Pack<T, V>, __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(p)));
  } else {
    q = *reinterpret_cast<const Pack<T, V>*>(p);
  }
  return q;
}
template <typename T, int V> __device__ __forceinline__ void store_nt(T* p, const float (&v)[V]) {
  constexpr int B = sizeof(T) * V;
  Pack<T, V> q;
#pragma unroll
  for (int e = 0; e < V; ++e) q.e[e] = (T)v[e];
  if constexpr (B >= 16) {
    struct Q { u32x4 w[B / 16]; };
    const Q u = __builtin_bit_cast(Q, q);
#pragma unroll
    for (int k = 0; k < B / 16; ++k) __builtin_nontemporal_store(u.w[k], reinterpret_cast<u32x4*>(p) + k);
  } else if constexpr (B == 8) {
    __builtin_nontemporal_store(__builtin_bit_cast(u32x2, q), reinterpret_cast<u32x2*>(p));
  } else if constexpr (B == 4) {
    __builtin_nontemporal_store(__builtin_bit_cast(uint32_t, q), reinterpret_cast<uint32_t*>(p));
  } else {
    *reinterpret_cast<Pack<T, V>*>(p) = q;
  }
}
template <bool NT, typename T, int V> __device__ __forceinline__ Pack<T, V> load_p(const T* p) {
  if constexpr (NT) return load_nt<T, V>(p);
  else return *reinterpret_cast<const Pack<T, V>*>(p);
}
template <bool NT, typename T, int V> __device__ __forceinline__ void store_p(T* p, const float (&v)[V]) {
  if constexpr (NT) store_nt<T, V>(p, v);
  else store_v<T, V>(p, v);
}

// Hides from the compiler that a register still holds what it held: it would otherwise keep a 16-bit vector's float32 form from one pass
// over the registers to the next, at twice the registers (18 vectors a thread spill then).
template <typename T, int V> __device__ __forceinline__ void keep_packed(Pack<T, V>& q) {
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
    struct Words { uint32_t w[V / 2]; };
    Words u = __builtin_bit_cast(Words, q);
#pragma unroll
    for (int e = 0; e < V / 2; ++e) asm volatile("" : "+v"(u.w[e]));
    q = __builtin_bit_cast(Pack<T, V>, u);
  }
}

// ---- activations ----
__device__ __forceinline__ float sigmoid_f(float z) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * z)); }
// The normal distribution's Phi(-|z|) = erfc(|z| / sqrt 2) / 2 by Abramowitz and Stegun 7.1.26 (a polynomial of the fifth degree in
// t = 1 / (1 + 0.3275911 |z| / sqrt 2) times exp(-z^2 / 2), 0.75e-7 off at the most, and as much again by rounding): 9 operations beside one
// exponential, which the gradient needs anyway, and one reciprocal; the library's erf is over twice that.  Halved coefficients.
__device__ __forceinline__ float phi_tail(float z, float gauss) {
  const float t = __builtin_amdgcn_rcpf(1.f + 0.23164189f * fabsf(z));
  return t * (0.127414796f + t * (-0.142248368f + t * (0.7107068705f + t * (-0.7265760135f + t * 0.5307027145f)))) * gauss;
}
__device__ __forceinline__ float gauss_f(float z) { return __builtin_amdgcn_exp2f(-0.72134752f * z * z); }
template <int V> __device__ __forceinline__ void act_apply(float (&z)[V], int act) {
  if (act == NORM_ACT_RELU) {
#pragma unroll
    for (int e = 0; e < V; ++e) z[e] = z[e] < 0.f ? 0.f : z[e];          // NaN stays (a maximum with zero would drop it)
  } else if (act == NORM_ACT_SILU) {
#pragma unroll
    for (int e = 0; e < V; ++e) z[e] *= sigmoid_f(z[e]);
  } else if (act == NORM_ACT_GELU) {
#pragma unroll
    for (int e = 0; e < V; ++e) z[e] = fmaxf(z[e], 0.f) - fabsf(z[e]) * phi_tail(z[e], gauss_f(z[e]));      // z Phi(z) on either side
  }
}
// g[e] *= act'(z[e])
template <int V> __device__ __forceinline__ void act_grad_apply(float (&g)[V], const float (&z)[V], int act) {
  if (act == NORM_ACT_RELU) {
#pragma unroll
    for (int e = 0; e < V; ++e) g[e] = z[e] <= 0.f ? 0.f : g[e];
  } else if (act == NORM_ACT_SILU) {
#pragma unroll
    for (int e = 0; e < V; ++e) { const float s = sigmoid_f(z[e]); g[e] *= s * (1.f + z[e] * (1.f - s)); }
  } else if (act == NORM_ACT_GELU) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float n = gauss_f(z[e]), q = phi_tail(z[e], n);
      g[e] *= (z[e] < 0.f ? q : 1.f - q) + z[e] * (0.39894228f * n);
    }
  }
}

// ---- arguments and tiles -----------------------------------------------------------------------------------------------------
// Every kernel below lets a thread keep one vector of V channels (column `col` of its workgroup's) and walk pixels: rows x cb threads.
struct NormArgs {
  const void* x; const void* dy; void* y;              // y: the output (dx in the backward pass)
  const float* gamma; const float* beta;               // nullable
  float* mean; float* rstd;                            // [N][G]
  float2* part;                                        // partial numbers of chunks: see the kernels
  float2* ab; float2* s12;                             // backward: (A, B) by channel, (S1, S2) / (P D) by group
  float* dgamma; float* dbeta;
  size_t xcs, ycs, dycs;                               // pixel strides, elements
  int n, p, c, groups, d;
  int cb, rows, span;                                  // columns and rows of a workgroup's threads, its channels
  int chunks, ppc;                                     // chunks of an image's pixels, pixels of a chunk: chunks = ceil(p / ppc)
  int achunks, appc;                                   // ... in the second of two launches
  int slots, per_group, jl;                            // see team_sums
  uint32_t by_d, by_cb, by_rows, by_per_group;               // for div_by
  float eps; int act, accumulate, team;                // team: the host's variant of the one-launch form
  DropArgs drop;
};
// x / y for x < 2^16 and y <= 2^16 by the host's ceil(2^32 / y) (0 for y = 1): a division by a number of the launch is some 20 instructions
// otherwise, as many as the work on three channels.
__device__ __forceinline__ int div_by(int x, uint32_t magic) { return magic ? (int)__umulhi((uint32_t)x, magic) : x; }
__device__ __forceinline__ uint64_t drop_offset(const DropArgs& d) { return d.offset + (d.counter ? *d.counter : 0); }
__device__ __forceinline__ float inv_std(float var, float eps) { return 1.f / sqrtf(var + eps); }

struct NormTeam {
  int img, cbase, row, col, c0;
  bool on;
};
template <int V> __device__ __forceinline__ void team_threads(NormTeam& t, const NormArgs& a) {
  t.row = div_by(threadIdx.x, a.by_cb);
  t.col = threadIdx.x - t.row * a.cb;
  t.c0 = t.cbase + t.col * V;
  t.on = t.row < a.rows;
}

// ---- sums over a workgroup's pixels and the channels of each of its groups: tot[group], seen by every thread.  All threads call. ----
// A thread first adds the channels of its vector that share a group (slots numbers are left: 1, V / d or V), a wave its rows where columns
// are a power of two, then 2^jl lanes a group add what is left of all groups at once.  `red`: TH * V floats.
template <int V> __device__ __forceinline__ int fold_slots(const NormArgs& a, float (&v)[V]) {
  if (a.slots < V) {                                         // (groups of one channel or of no divisor's fraction of V stay as they are)
#pragma unroll
    for (int k = V; k > 1; k >>= 1)
      if (a.slots < k) {
#pragma unroll
        for (int e = 0; e < k / 2; ++e) v[e] = v[2 * e] + v[2 * e + 1];
      }
  }
  return a.slots;
}
template <int V, int TH> __device__ __forceinline__ void team_sums(const NormArgs& a, const NormTeam& t, float (&v)[V], float* red, float* tot) {
  const int slots = fold_slots<V>(a, v), per_row = a.cb * slots;
  const bool pow2 = a.cb <= 64 && (a.cb & (a.cb - 1)) == 0;
  int rows = a.rows;
  if (pow2) {
    rows = TH / 64;
    for (int k = a.cb; k < 64; k <<= 1) {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e < slots) v[e] += __shfl_xor(v[e], k);
    }
  }
  const int r = pow2 ? threadIdx.x >> 6 : t.row;
  if (pow2 ? (int)(threadIdx.x & 63) < a.cb : t.on) {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < slots) red[r * per_row + t.col * slots + e] = v[e];
  }
  __syncthreads();
  const int lanes = 1 << a.jl, lane = threadIdx.x & (lanes - 1), groups = a.span / a.d, total = rows * a.per_group;
  for (int j0 = 0; j0 < groups; j0 += TH >> a.jl) {          // (every lane of a wave takes part in the shuffles)
    const int j = j0 + (threadIdx.x >> a.jl);
    float s = 0.f;
    if (j < groups)
      for (int i = lane; i < total; i += lanes) { const int q = div_by(i, a.by_per_group); s += red[q * per_row + j * a.per_group + (i - q * a.per_group)]; }
    for (int k = lanes >> 1; k; k >>= 1) s += __shfl_xor(s, k);
    if (j < groups && lane == 0) tot[j] = s;
  }
  __syncthreads();
}

// ---- one launch, one read: a workgroup holds `span` channels (whole groups) of all pixels of an image in registers ----
// Thread (row, col) keeps the vectors of column col at the pixels row + r * rows, r < R, as they were loaded (16-bit tensors packed).
// What a second pass over memory would be is a pass over registers, so the mean comes first and the squares are about it.
// Workgroup b runs on XCD b % 8 (observed; speed only): the workgroups of one image, which share its cache lines where a span is less than a
// line, go to one XCD.
template <int V> __device__ __forceinline__ NormTeam span_team(const NormArgs& a) {
  NormTeam t;
  const int slices = a.c / a.span, b = blockIdx.x, whole = a.n / 8 * 8 * slices;
  int unit = b;
  if (b < whole) { const int k = b >> 3; unit = (k / slices * 8 + (b & 7)) * slices + k % slices; }
  t.img = unit / slices;
  t.cbase = (unit - t.img * slices) * a.span;
  team_threads<V>(t, a);
  return t;
}

template <typename T, int V, int R, int TH> __global__ __launch_bounds__(TH) void norm_team_kernel(const NormArgs a) {
  __shared__ float red[TH * V];
  __shared__ float tot[2][TH * V];                           // (as many groups as channels at the most)
  const NormTeam t = span_team<V>(a);
  const T* x = (const T*)a.x + (size_t)t.img * a.p * a.xcs + t.c0;
  Pack<T, V> q[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int p = t.row + r * a.rows;
    if (t.on && p < a.p) q[r] = *reinterpret_cast<const Pack<T, V>*>(x + (size_t)p * a.xcs);
  }
  float gamma[V], beta[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    gamma[e] = t.on && a.gamma ? a.gamma[t.c0 + e] : 1.f;
    beta[e] = t.on && a.beta ? a.beta[t.c0 + e] : 0.f;
  }
  float s[V];
#pragma unroll
  for (int e = 0; e < V; ++e) s[e] = 0.f;
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (t.on && t.row + r * a.rows < a.p) {
#pragma unroll
      for (int e = 0; e < V; ++e) s[e] += (float)q[r].e[e];
    }
  team_sums<V, TH>(a, t, s, red, tot[0]);
#pragma unroll
  for (int r = 0; r < R; ++r) keep_packed<T, V>(q[r]);
  const float inv = 1.f / ((float)a.p * (float)a.d);
  float mean[V];
#pragma unroll
  for (int e = 0; e < V; ++e) { mean[e] = t.on ? tot[0][div_by(t.col * V + e, a.by_d)] * inv : 0.f; s[e] = 0.f; }
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (t.on && t.row + r * a.rows < a.p) {
#pragma unroll
      for (int e = 0; e < V; ++e) { const float dv = (float)q[r].e[e] - mean[e]; s[e] += dv * dv; }
    }
  team_sums<V, TH>(a, t, s, red, tot[1]);
#pragma unroll
  for (int r = 0; r < R; ++r) keep_packed<T, V>(q[r]);
  for (int j = threadIdx.x; j < a.span / a.d; j += TH) {
    const size_t g = (size_t)t.img * a.groups + t.cbase / a.d + j;
    a.mean[g] = tot[0][j] * inv;
    a.rstd[g] = inv_std(tot[1][j] * inv, a.eps);
  }
  if (!t.on) return;
#pragma unroll
  for (int e = 0; e < V; ++e) gamma[e] *= inv_std(tot[1][div_by(t.col * V + e, a.by_d)] * inv, a.eps);
  const uint64_t offset = a.drop.thresh ? drop_offset(a.drop) : 0;
  T* y = (T*)a.y + (size_t)t.img * a.p * a.ycs + t.c0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int p = t.row + r * a.rows;
    if (p < a.p) {
      float v[V];
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = ((float)q[r].e[e] - mean[e]) * gamma[e] + beta[e];
      act_apply<V>(v, a.act);
      if (a.drop.thresh) drop_apply<V>(v, ((uint64_t)t.img * a.p + p) * a.c + t.c0, a.drop, offset);
      store_v<T, V>(y + (size_t)p * a.ycs, v);
    }
  }
}

// ---- two launches, one read each: statistics per group and chunk of pixels, then the output ----
// part[image][group][chunk] = (mean, M2) of a chunk.  The second launch's workgroups join their image's chunks themselves, or, where that is
// much to read for each of them (few images with many chunks), norm_join_kernel joins them once in between.
template <int V> __device__ __forceinline__ NormTeam chunk_team(const NormArgs& a, int block, int chunks, int ppc, int& chunk, int& p0, int& p1) {
  NormTeam t;
  t.img = block / chunks;
  chunk = block - t.img * chunks;
  p0 = chunk * ppc; p1 = min(a.p, p0 + ppc);
  t.cbase = blockIdx.y * a.span;
  team_threads<V>(t, a);
  return t;
}

// One batch of M <= U pixels joined to the running (mean, M2) of the thread's channels: the batch is reduced about its own mean and joined by
// Chan's formula, so nothing is lost when the mean is large against the spread: no sum of squares about a far point exists anywhere.
template <typename T, int V, int U> __device__ __forceinline__ void stats_batch(Pack<T, V> (&q)[U], int m, float (&mean)[V], float (&m2)[V], float& cnt) {
  float bm[V], b2[V];
  const float fm = (float)m, im = 1.f / fm, w = fm / (cnt + fm), nw = cnt * w;
  cnt += fm;
#pragma unroll
  for (int e = 0; e < V; ++e) bm[e] = b2[e] = 0.f;
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (u < m) {
#pragma unroll
      for (int e = 0; e < V; ++e) bm[e] += (float)q[u].e[e];
    }
#pragma unroll
  for (int e = 0; e < V; ++e) bm[e] *= im;
#pragma unroll
  for (int u = 0; u < U; ++u) keep_packed<T, V>(q[u]);
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (u < m) {
#pragma unroll
      for (int e = 0; e < V; ++e) { const float dv = (float)q[u].e[e] - bm[e]; b2[e] += dv * dv; }
    }
#pragma unroll
  for (int e = 0; e < V; ++e) { const float dm = bm[e] - mean[e]; mean[e] += dm * w; m2[e] += b2[e] + dm * dm * nw; }
}

template <typename T, int V, int TH, bool NT> __global__ __launch_bounds__(TH) void norm_chunk_stats_kernel(const NormArgs a) {
  constexpr int U = 4;
  __shared__ float red[TH * V];
  __shared__ float tot[2][TH * V];
  int chunk, p0, p1;
  const NormTeam t = chunk_team<V>(a, blockIdx.x, a.chunks, a.ppc, chunk, p0, p1);
  float mean[V], m2[V], cnt = 0.f;
#pragma unroll
  for (int e = 0; e < V; ++e) mean[e] = m2[e] = 0.f;
  if (t.on) {
    const size_t step = (size_t)a.rows * a.xcs;
    const T* x = (const T*)a.x + ((size_t)t.img * a.p + p0 + t.row) * a.xcs + t.c0;
    const int batches = (p1 - p0) / (U * a.rows);            // full ones: the same for every thread
    Pack<T, V> q[U], next[U];
    if (batches) {
#pragma unroll
      for (int u = 0; u < U; ++u) next[u] = load_p<NT, T, V>(x + u * step);
    }
    for (int k = 0; k < batches; ++k) {                      // the next batch is on its way while this one is reduced
#pragma unroll
      for (int u = 0; u < U; ++u) q[u] = next[u];
      x += U * step;
      if (k + 1 < batches) {
#pragma unroll
        for (int u = 0; u < U; ++u) next[u] = load_p<NT, T, V>(x + u * step);
      }
      stats_batch<T, V, U>(q, U, mean, m2, cnt);
    }
    const int left = p1 - (p0 + t.row + batches * U * a.rows), m = left > 0 ? (left + a.rows - 1) / a.rows : 0;
    if (m) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (u < m) q[u] = load_p<NT, T, V>(x + u * step);
      stats_batch<T, V, U>(q, m, mean, m2, cnt);
    }
  }
  float s[V];
#pragma unroll
  for (int e = 0; e < V; ++e) s[e] = cnt * mean[e];
  team_sums<V, TH>(a, t, s, red, tot[0]);
  const float inv = 1.f / ((float)(p1 - p0) * (float)a.d);
#pragma unroll
  for (int e = 0; e < V; ++e) { const float dm = t.on ? mean[e] - tot[0][div_by(t.col * V + e, a.by_d)] * inv : 0.f; s[e] = m2[e] + cnt * dm * dm; }
  team_sums<V, TH>(a, t, s, red, tot[1]);
  for (int j = threadIdx.x; j < a.span / a.d; j += TH)
    a.part[((size_t)t.img * a.groups + t.cbase / a.d + j) * a.chunks + chunk] = make_float2(tot[0][j] * inv, tot[1][j]);
}

// mean and rstd of `count` groups from the chunks' numbers: 2^jl lanes a group, all groups at once (a wave a group in turn would be two round
// trips to memory for every group after the other: 10 us for 32 groups)
// Up to K numbers a lane stay in registers between the two sums: one trip to memory.
template <int TH, int K> __device__ __forceinline__ void join_groups(const NormArgs& a, size_t first, int count, float* mean, float* rstd) {
  const int lanes = 1 << a.jl, lane = threadIdx.x & (lanes - 1);
  const float m = (float)a.p * (float)a.d, full = (float)a.ppc * (float)a.d, last = (float)(a.p - (a.chunks - 1) * a.ppc) * (float)a.d;
  for (int j0 = 0; j0 < count; j0 += TH >> a.jl) {
    const int j = j0 + (threadIdx.x >> a.jl);
    const float2* part = a.part + (first + j) * a.chunks;
    float2 f[K];
    float s = 0.f, q = 0.f;
    if (j < count) {
#pragma unroll
      for (int i = 0; i < K; ++i) f[i] = lane + i * lanes < a.chunks ? part[lane + i * lanes] : make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < K; ++i) s += f[i].x * (lane + i * lanes == a.chunks - 1 ? last : full);
      for (int k = lane + K * lanes; k < a.chunks; k += lanes) s += part[k].x * (k == a.chunks - 1 ? last : full);
    }
    for (int k = lanes >> 1; k; k >>= 1) s += __shfl_xor(s, k);
    const float mu = s / m;
    if (j < count) {
#pragma unroll
      for (int i = 0; i < K; ++i)
        if (lane + i * lanes < a.chunks) q += f[i].y + (f[i].x - mu) * (f[i].x - mu) * (lane + i * lanes == a.chunks - 1 ? last : full);
      for (int k = lane + K * lanes; k < a.chunks; k += lanes) {
        const float2 g = part[k];
        q += g.y + (g.x - mu) * (g.x - mu) * (k == a.chunks - 1 ? last : full);
      }
    }
    for (int k = lanes >> 1; k; k >>= 1) q += __shfl_xor(q, k);
    if (j < count && lane == 0) { mean[j] = mu; rstd[j] = inv_std(q / m, a.eps); }
  }
}
// a wave a group of the whole batch (jl = 6)
__global__ __launch_bounds__(64) void norm_join_kernel(const NormArgs a) {
  join_groups<64, 16>(a, blockIdx.x, 1, a.mean + blockIdx.x, a.rstd + blockIdx.x);
}

// Two pixels' dropout of a thread with four channels: a generator block is eight, so lanes 2k and 2k + 1 want the same two blocks.  Each
// computes one and they exchange halves.  The span's channels are a multiple of 8, so both lanes are at the same pixels.
template <int V> __device__ __forceinline__ void drop_apply_pair(float (&v0)[V], float (&v1)[V], uint64_t i0, uint64_t i1, const DropArgs& d, uint64_t offset) {
  static_assert(V == 4, "");
  const bool odd = threadIdx.x & 1;
  const Philox r = philox7((odd ? i1 : i0) >> 3, offset, d.seed);
  const uint32_t s0 = odd ? r.w[0] : r.w[2], s1 = odd ? r.w[1] : r.w[3];
  const uint32_t g0 = __builtin_amdgcn_mov_dpp(s0, 0xB1, 0xf, 0xf, true), g1 = __builtin_amdgcn_mov_dpp(s1, 0xB1, 0xf, 0xf, true);   // quad_perm 1, 0, 3, 2
  const uint32_t a0 = odd ? g0 : r.w[0], a1 = odd ? g1 : r.w[1], b0 = odd ? r.w[2] : g0, b1 = odd ? r.w[3] : g1;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const uint32_t wa = e & 2 ? a1 : a0, wb = e & 2 ? b1 : b0;
    v0[e] = (e & 1 ? wa >> 16 : wa & 0xffffu) >= d.thresh ? v0[e] * d.scale : 0.f;
    v1[e] = (e & 1 ? wb >> 16 : wb & 0xffffu) >= d.thresh ? v1[e] * d.scale : 0.f;
  }
}

// U pixels of a thread from pixel p on, m of them there
template <typename T, int V, int U, bool NT> __device__ __forceinline__ void load_batch(Pack<T, V> (&q)[U], const T* base, size_t cs, int rows, int p, int m) {
  const T* x = base + (size_t)p * cs;
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (u < m) q[u] = load_p<NT, T, V>(x + (size_t)(u * rows) * cs);
}
__device__ __forceinline__ int batch_count(const NormArgs& a, const NormTeam& t, int p, int p1) { return t.on && p < p1 ? div_by(min(p1 - p, 65535 - a.rows) + a.rows - 1, a.by_rows) : 0; }

template <typename T, int V, int TH, bool NT> __global__ __launch_bounds__(TH) void norm_chunk_apply_kernel(const NormArgs a, int join) {
  constexpr int U = 4;
  __shared__ float mean_s[TH * V], rstd_s[TH * V];
  int chunk, p0, p1;
  const NormTeam t = chunk_team<V>(a, blockIdx.x, a.achunks, a.appc, chunk, p0, p1);
  const T* x = (const T*)a.x + (size_t)t.img * a.p * a.xcs + t.c0;
  T* y = (T*)a.y + (size_t)t.img * a.p * a.ycs + t.c0;
  int p = p0 + t.row, m = batch_count(a, t, p, p1);
  Pack<T, V> q[U], next[U];
  load_batch<T, V, U, NT>(q, x, a.xcs, a.rows, p, m);        // on its way while the statistics come
  const size_t g0 = (size_t)t.img * a.groups + div_by(t.cbase, a.by_d);
  const float *mg = a.mean + g0, *rg = a.rstd + g0;
  float mean[V], scale[V], beta[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    scale[e] = t.on && a.gamma ? a.gamma[t.c0 + e] : 1.f;
    beta[e] = t.on && a.beta ? a.beta[t.c0 + e] : 0.f;
  }
  if (join) {
    const int groups = div_by(a.span, a.by_d);
    join_groups<TH, 4>(a, g0, groups, mean_s, rstd_s);
    __syncthreads();
    if (chunk == 0)
      for (int j = threadIdx.x; j < groups; j += TH) { a.mean[g0 + j] = mean_s[j]; a.rstd[g0 + j] = rstd_s[j]; }
  }
  if (!t.on) return;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const int g = div_by(t.col * V + e, a.by_d);
    mean[e] = join ? mean_s[g] : mg[g];
    scale[e] *= join ? rstd_s[g] : rg[g];
  }
  const uint64_t offset = a.drop.thresh ? drop_offset(a.drop) : 0;
  const bool pairs = V == 4 && a.span % 8 == 0;
  while (m) {
    const int pn = p + U * a.rows, mn = batch_count(a, t, pn, p1);
    load_batch<T, V, U, NT>(next, x, a.xcs, a.rows, pn, mn);
    const uint64_t i = ((uint64_t)t.img * a.p + p) * a.c + t.c0, di = (uint64_t)a.rows * a.c;
#pragma unroll
    for (int u = 0; u < U; u += 2) {
      float v[2][V];
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (u + k < m) {
#pragma unroll
          for (int e = 0; e < V; ++e) v[k][e] = ((float)q[u + k].e[e] - mean[e]) * scale[e] + beta[e];
          act_apply<V>(v[k], a.act);
          if (a.drop.thresh && !pairs) drop_apply<V>(v[k], i + (u + k) * di, a.drop, offset);
        }
      if constexpr (V == 4) {
        if (a.drop.thresh && pairs && u < m) drop_apply_pair<V>(v[0], v[1], i + u * di, i + (u + 1) * di, a.drop, offset);   // (the second may be no pixel: not stored)
      }
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (u + k < m) store_p<true, T, V>(y + (size_t)(p + (u + k) * a.rows) * a.ycs, v[k]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) q[u] = next[u];
    p = pn; m = mn;
  }
}

// ---- backward ----
// What a thread needs of its channels: xh = (x - mean) * rstd, z = xh * gamma + beta.
template <int V> struct NormChan {
  float mean[V], rstd[V], gamma[V], beta[V];
  __device__ __forceinline__ void load(const NormArgs& a, int img, int c0, bool on) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const size_t g = (size_t)img * a.groups + (on ? div_by(c0 + e, a.by_d) : 0);
      mean[e] = a.mean[g];
      rstd[e] = a.rstd[g];
      gamma[e] = on && a.gamma ? a.gamma[c0 + e] : 1.f;
      beta[e] = on && a.beta ? a.beta[c0 + e] : 0.f;
    }
  }
};
// v: x -> xh; g: dy (already dropped) -> dz
template <int V> __device__ __forceinline__ void norm_dz(const NormArgs& a, const NormChan<V>& ch, float (&v)[V], float (&g)[V]) {
  float z[V];
#pragma unroll
  for (int e = 0; e < V; ++e) { v[e] = (v[e] - ch.mean[e]) * ch.rstd[e]; z[e] = v[e] * ch.gamma[e] + ch.beta[e]; }
  act_grad_apply<V>(g, z, a.act);
}
// (A, B) of each of the workgroup's channels from its threads' sums, in sum[0 .. span), seen by every thread.  All threads call.
// sum: TH * V numbers.
template <int V, int TH> __device__ __forceinline__ void team_channels(const NormArgs& a, const NormTeam& t, float (&sa)[V], float (&sb)[V], float2* sum) {
  const bool pow2 = a.cb <= 64 && (a.cb & (a.cb - 1)) == 0;
  if (pow2)
    for (int k = a.cb; k < 64; k <<= 1) {
#pragma unroll
      for (int e = 0; e < V; ++e) { sa[e] += __shfl_xor(sa[e], k); sb[e] += __shfl_xor(sb[e], k); }
    }
  const int rows = pow2 ? TH / 64 : a.rows, r = pow2 ? threadIdx.x >> 6 : t.row;
  if (pow2 ? (int)(threadIdx.x & 63) < a.cb : t.on) {
#pragma unroll
    for (int e = 0; e < V; ++e) sum[r * a.span + t.col * V + e] = make_float2(sa[e], sb[e]);
  }
  __syncthreads();
  for (int c = threadIdx.x; c < a.span; c += TH) {
    float2 s = sum[c];
    for (int k = 1; k < rows; ++k) { const float2 f = sum[k * a.span + c]; s.x += f.x; s.y += f.y; }
    sum[c] = s;                                              // (a column is read and written by one thread)
  }
  __syncthreads();
}
// (sum of gamma A, sum of gamma B) * scale of each of the workgroup's groups.  All threads call.
template <int TH> __device__ __forceinline__ void team_group_sums(const NormArgs& a, const NormTeam& t, const float2* sum, float scale, float2* out) {
  const int lanes = 1 << a.jl, lane = threadIdx.x & (lanes - 1), groups = a.span / a.d;
  for (int j0 = 0; j0 < groups; j0 += TH >> a.jl) {
    const int j = j0 + (threadIdx.x >> a.jl);
    float s1 = 0.f, s2 = 0.f;
    if (j < groups)
      for (int k = lane; k < a.d; k += lanes) {
        const float2 f = sum[j * a.d + k];
        const float gm = a.gamma ? a.gamma[t.cbase + j * a.d + k] : 1.f;
        s1 += gm * f.x; s2 += gm * f.y;
      }
    for (int k = lanes >> 1; k; k >>= 1) { s1 += __shfl_xor(s1, k); s2 += __shfl_xor(s2, k); }
    if (j < groups && lane == 0) out[j] = make_float2(s1 * scale, s2 * scale);
  }
}

// The whole backward pass of a span in registers, x and dy read once: (A, B) of its channels go to ab[image][channel] for the parameters'
// gradients over the images.
template <typename T, int V, int R, int TH> __global__ __launch_bounds__(TH) void norm_team_grad_kernel(const NormArgs a) {
  __shared__ float2 sum[TH * V];
  __shared__ float2 tot[TH * V];
  const NormTeam t = span_team<V>(a);
  const T* x = (const T*)a.x + (size_t)t.img * a.p * a.xcs + t.c0;
  const T* dy = (const T*)a.dy + (size_t)t.img * a.p * a.dycs + t.c0;
  Pack<T, V> q[R], g[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int p = t.row + r * a.rows;
    if (t.on && p < a.p) {
      q[r] = *reinterpret_cast<const Pack<T, V>*>(x + (size_t)p * a.xcs);
      g[r] = *reinterpret_cast<const Pack<T, V>*>(dy + (size_t)p * a.dycs);
    }
  }
  NormChan<V> ch;
  ch.load(a, t.img, t.c0, t.on);
  const uint64_t offset = a.drop.thresh ? drop_offset(a.drop) : 0;
  float sa[V], sb[V];
#pragma unroll
  for (int e = 0; e < V; ++e) sa[e] = sb[e] = 0.f;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int p = t.row + r * a.rows;
    if (t.on && p < a.p) {
      float v[V], w[V];
      widen<T, V>(q[r], v);
      widen<T, V>(g[r], w);
      if (a.drop.thresh) drop_apply<V>(w, ((uint64_t)t.img * a.p + p) * a.c + t.c0, a.drop, offset);
      norm_dz<V>(a, ch, v, w);
#pragma unroll
      for (int e = 0; e < V; ++e) { sa[e] += w[e]; sb[e] += w[e] * v[e]; }
    }
  }
  team_channels<V, TH>(a, t, sa, sb, sum);
  team_group_sums<TH>(a, t, sum, 1.f / ((float)a.p * (float)a.d), tot);
  for (int c = threadIdx.x; c < a.span; c += TH) a.ab[(size_t)t.img * a.c + t.cbase + c] = sum[c];
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) { keep_packed<T, V>(q[r]); keep_packed<T, V>(g[r]); }
  if (!t.on) return;
  T* dx = (T*)a.y + (size_t)t.img * a.p * a.ycs + t.c0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int p = t.row + r * a.rows;
    if (p < a.p) {
      float v[V], w[V];
      widen<T, V>(q[r], v);
      widen<T, V>(g[r], w);
      if (a.drop.thresh) drop_apply<V>(w, ((uint64_t)t.img * a.p + p) * a.c + t.c0, a.drop, offset);
      norm_dz<V>(a, ch, v, w);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float2 s = tot[div_by(t.col * V + e, a.by_d)];
        w[e] = ch.rstd[e] * (w[e] * ch.gamma[e] - s.x - v[e] * s.y);
      }
      store_v<T, V>(dx + (size_t)p * a.ycs, w);
    }
  }
}

// dz (w) and xh (v) of the K pixels p, p + rows .. of the two-launch form from packed x and dy; K = 2 where a generator block is two
// threads' work, m of them there
template <typename T, int V> struct GradPixels {
  static constexpr int K = V == 4 ? 2 : 1;
  float v[K][V], w[K][V];
  __device__ __forceinline__ void get(const NormArgs& a, const NormTeam& t, const NormChan<V>& ch, const Pack<T, V>* q, const Pack<T, V>* g, int p, int m,
                                      uint64_t offset) {
    const uint64_t i = ((uint64_t)t.img * a.p + p) * a.c + t.c0, di = (uint64_t)a.rows * a.c;
    bool pairs = false;
#pragma unroll
    for (int k = 0; k < K; ++k) { widen<T, V>(q[k], v[k]); widen<T, V>(g[k], w[k]); }
    if constexpr (K == 2) {
      pairs = a.span % 8 == 0;
      if (a.drop.thresh && pairs) drop_apply_pair<V>(w[0], w[1], i, i + di, a.drop, offset);
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (k < m) {
        if (a.drop.thresh && !pairs) drop_apply<V>(w[k], i + k * di, a.drop, offset);
        norm_dz<V>(a, ch, v[k], w[k]);
      }
  }
};

// First launch: part[image][chunk][channel] = (A, B) of a chunk, and behind it s12[image][group][chunk] = (sum of gamma A, of gamma B) / (P D).
template <typename T, int V, int TH, bool NT> __global__ __launch_bounds__(TH) void norm_chunk_sums_kernel(const NormArgs a) {
  constexpr int U = sizeof(T) * V == 8 ? 4 : 2;
  __shared__ float2 sum[TH * V];
  __shared__ float2 tot[TH * V];
  int chunk, p0, p1;
  const NormTeam t = chunk_team<V>(a, blockIdx.x, a.chunks, a.ppc, chunk, p0, p1);
  const T* x = (const T*)a.x + (size_t)t.img * a.p * a.xcs + t.c0;
  const T* dy = (const T*)a.dy + (size_t)t.img * a.p * a.dycs + t.c0;
  int p = p0 + t.row, m = batch_count(a, t, p, p1);
  Pack<T, V> q[U], g[U], nq[U], ng[U];
  load_batch<T, V, U, NT>(q, x, a.xcs, a.rows, p, m);
  load_batch<T, V, U, NT>(g, dy, a.dycs, a.rows, p, m);
  NormChan<V> ch;
  ch.load(a, t.img, t.c0, t.on);
  const uint64_t offset = a.drop.thresh ? drop_offset(a.drop) : 0;
  float sa[V], sb[V];
#pragma unroll
  for (int e = 0; e < V; ++e) sa[e] = sb[e] = 0.f;
  while (m) {
    const int pn = p + U * a.rows, mn = batch_count(a, t, pn, p1);
    load_batch<T, V, U, NT>(nq, x, a.xcs, a.rows, pn, mn);
    load_batch<T, V, U, NT>(ng, dy, a.dycs, a.rows, pn, mn);
#pragma unroll
    for (int u = 0; u < U; u += GradPixels<T, V>::K)
      if (u < m) {
        GradPixels<T, V> b;
        b.get(a, t, ch, q + u, g + u, p + u * a.rows, m - u, offset);
#pragma unroll
        for (int k = 0; k < GradPixels<T, V>::K; ++k)
          if (u + k < m) {
#pragma unroll
            for (int e = 0; e < V; ++e) { sa[e] += b.w[k][e]; sb[e] += b.w[k][e] * b.v[k][e]; }
          }
      }
#pragma unroll
    for (int u = 0; u < U; ++u) { q[u] = nq[u]; g[u] = ng[u]; }
    p = pn; m = mn;
  }
  team_channels<V, TH>(a, t, sa, sb, sum);
  team_group_sums<TH>(a, t, sum, 1.f / ((float)a.p * (float)a.d), tot);
  for (int c = threadIdx.x; c < a.span; c += TH) a.part[((size_t)t.img * a.chunks + chunk) * a.c + t.cbase + c] = sum[c];
  __syncthreads();
  for (int j = threadIdx.x; j < a.span / a.d; j += TH) a.s12[((size_t)t.img * a.groups + t.cbase / a.d + j) * a.chunks + chunk] = tot[j];
}

// dgamma, dbeta of 16 channels: the sum over `rows` rows of (A, B) by channel (float64: a row is a chunk's or an image's sum)
__device__ __forceinline__ void param_grads(const NormArgs& a, const float2* ab, int rows, int block) {
  __shared__ double2 red[256];
  const int ch = block * 16 + (threadIdx.x & 15);
  double sa = 0.0, sb = 0.0;
  if (ch < a.c) {
#pragma unroll 4
    for (int r = threadIdx.x >> 4; r < rows; r += 16) { const float2 f = ab[(size_t)r * a.c + ch]; sa += f.x; sb += f.y; }
  }
  red[threadIdx.x] = make_double2(sa, sb);
  __syncthreads();
  if (threadIdx.x < 16 && ch < a.c) {
    for (int k = 1; k < 16; ++k) { sa += red[16 * k + threadIdx.x].x; sb += red[16 * k + threadIdx.x].y; }
    if (a.dbeta) a.dbeta[ch] = (float)(a.accumulate ? a.dbeta[ch] + sa : sa);
    if (a.dgamma) a.dgamma[ch] = (float)(a.accumulate ? a.dgamma[ch] + sb : sb);
  }
}
__global__ __launch_bounds__(256) void norm_params_kernel(const NormArgs a, const float2* ab, int rows) { param_grads(a, ab, rows, blockIdx.x); }

// Second launch: dx.  Its first `pblocks` workgroups sum the parameters' gradients instead.
template <typename T, int V, int TH, bool NT> __global__ __launch_bounds__(TH) void norm_chunk_grad_kernel(const NormArgs a, int pblocks) {
  static_assert(TH == 256, "param_grads");
  constexpr int U = sizeof(T) * V == 8 ? 4 : 2;
  __shared__ float2 tot[TH * V];
  if ((int)blockIdx.x < pblocks) {
    if (blockIdx.y == 0) param_grads(a, a.part, a.n * a.chunks, blockIdx.x);
    return;
  }
  int chunk, p0, p1;
  const NormTeam t = chunk_team<V>(a, blockIdx.x - pblocks, a.achunks, a.appc, chunk, p0, p1);
  const T* x = (const T*)a.x + (size_t)t.img * a.p * a.xcs + t.c0;
  const T* dy = (const T*)a.dy + (size_t)t.img * a.p * a.dycs + t.c0;
  int p = p0 + t.row, m = batch_count(a, t, p, p1);
  Pack<T, V> q[U], g[U], nq[U], ng[U];
  load_batch<T, V, U, NT>(q, x, a.xcs, a.rows, p, m);
  load_batch<T, V, U, NT>(g, dy, a.dycs, a.rows, p, m);
  NormChan<V> ch;
  ch.load(a, t.img, t.c0, t.on);
  {
    const int lanes = 1 << a.jl, lane = threadIdx.x & (lanes - 1), groups = a.span / a.d;
    for (int j0 = 0; j0 < groups; j0 += TH >> a.jl) {
      const int j = j0 + (threadIdx.x >> a.jl);
      float s1 = 0.f, s2 = 0.f;
      if (j < groups) {
        const float2* part = a.s12 + ((size_t)t.img * a.groups + t.cbase / a.d + j) * a.chunks;
#pragma unroll 4
        for (int k = lane; k < a.chunks; k += lanes) { const float2 f = part[k]; s1 += f.x; s2 += f.y; }
      }
      for (int k = lanes >> 1; k; k >>= 1) { s1 += __shfl_xor(s1, k); s2 += __shfl_xor(s2, k); }
      if (j < groups && lane == 0) tot[j] = make_float2(s1, s2);
    }
    __syncthreads();
  }
  if (!t.on) return;
  T* dx = (T*)a.y + (size_t)t.img * a.p * a.ycs + t.c0;
  float s1[V], s2[V];
#pragma unroll
  for (int e = 0; e < V; ++e) { const float2 s = tot[div_by(t.col * V + e, a.by_d)]; s1[e] = s.x; s2[e] = s.y; }
  const uint64_t offset = a.drop.thresh ? drop_offset(a.drop) : 0;
  while (m) {
    const int pn = p + U * a.rows, mn = batch_count(a, t, pn, p1);
    load_batch<T, V, U, NT>(nq, x, a.xcs, a.rows, pn, mn);
    load_batch<T, V, U, NT>(ng, dy, a.dycs, a.rows, pn, mn);
#pragma unroll
    for (int u = 0; u < U; u += GradPixels<T, V>::K)
      if (u < m) {
        GradPixels<T, V> b;
        b.get(a, t, ch, q + u, g + u, p + u * a.rows, m - u, offset);
#pragma unroll
        for (int k = 0; k < GradPixels<T, V>::K; ++k)
          if (u + k < m) {
#pragma unroll
            for (int e = 0; e < V; ++e) b.w[k][e] = ch.rstd[e] * (b.w[k][e] * ch.gamma[e] - s1[e] - b.v[k][e] * s2[e]);
            store_p<true, T, V>(dx + (size_t)(p + (u + k) * a.rows) * a.ycs, b.w[k]);
          }
      }
#pragma unroll
    for (int u = 0; u < U; ++u) { q[u] = nq[u]; g[u] = ng[u]; }
    p = pn; m = mn;
  }
}

// ---- any shape: workgroups of any channels, three launches (four backward).  What the forms above do not take: pixels of more vectors
// than a workgroup has threads ----
struct NormTile {
  int img, chunk, p0, p1, row, c0;
  bool on;
  template <int V> __device__ __forceinline__ static NormTile get(const NormArgs& a) {
    NormTile t;
    t.img = blockIdx.x / a.chunks; t.chunk = blockIdx.x - t.img * a.chunks;
    t.p0 = t.chunk * a.ppc; t.p1 = min(a.p, t.p0 + a.ppc);
    t.row = threadIdx.x / a.cb;
    t.c0 = (blockIdx.y * a.cb + (threadIdx.x - t.row * a.cb)) * V;
    t.on = t.row < a.rows && t.c0 < a.c;
    return t;
  }
};

// ---- statistics, first half: (mean, M2) of every channel over a chunk ----
template <typename T, int V> __global__ __launch_bounds__(256) void norm_stats_kernel(const NormArgs a) {
  constexpr int U = 4;
  __shared__ float2 red[256 * V];
  const NormTile t = NormTile::get<V>(a);
  float mean[V], m2[V];
#pragma unroll
  for (int e = 0; e < V; ++e) mean[e] = m2[e] = 0.f;
  if (t.on) {
    const T* x = (const T*)a.x + ((size_t)t.img * a.p) * a.xcs + t.c0;
    float cnt = 0.f;
    for (int p = t.p0 + t.row; p < t.p1; p += U * a.rows) {
      const int m = min(U, (t.p1 - p + a.rows - 1) / a.rows);
      Pack<T, V> q[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (u < m) q[u] = load_p<false, T, V>(x + (size_t)(p + u * a.rows) * a.xcs);
      stats_batch<T, V, U>(q, m, mean, m2, cnt);
    }
#pragma unroll
    for (int e = 0; e < V; ++e) red[threadIdx.x * V + e] = make_float2(mean[e], m2[e]);
  }
  __syncthreads();
  const int len = t.p1 - t.p0, nch = min(a.cb * V, a.c - (int)blockIdx.y * a.cb * V);
  for (int ch = threadIdx.x; ch < nch; ch += 256) {
    float s = 0.f;
    for (int r = 0; r < min(a.rows, len); ++r) s += red[r * a.cb * V + ch].x * (float)((len - r + a.rows - 1) / a.rows);
    const float m = s / (float)len;
    float q = 0.f;
    for (int r = 0; r < min(a.rows, len); ++r) {
      const float2 f = red[r * a.cb * V + ch];
      q += f.y + (float)((len - r + a.rows - 1) / a.rows) * (f.x - m) * (f.x - m);
    }
    a.part[((size_t)t.img * a.chunks + t.chunk) * a.c + blockIdx.y * a.cb * V + ch] = make_float2(m, q);
  }
}

__device__ __forceinline__ double block_sum(double v, double* red) {            // 256 threads; the same value for every thread
#pragma unroll
  for (int s = 32; s; s >>= 1) v += __shfl_xor(v, s);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

// ---- statistics, second half: one workgroup per (image, group) joins the chunks' (mean, M2) of its channels ----
__global__ __launch_bounds__(256) void norm_stats_join_kernel(const NormArgs a) {
  __shared__ double red[4];
  const int img = blockIdx.x / a.groups, g = blockIdx.x - img * a.groups;
  const float2* part = a.part + (size_t)img * a.chunks * a.c + (size_t)g * a.d;
  const int total = a.chunks * a.d;
  const double m = (double)a.p * a.d;
  double s = 0.0;
  for (int i = threadIdx.x; i < total; i += 256) {
    const int k = i / a.d, ch = i - k * a.d;
    s += (double)part[(size_t)k * a.c + ch].x * min(a.ppc, a.p - k * a.ppc);
  }
  const double mean = block_sum(s, red) / m;
  double q = 0.0;
  for (int i = threadIdx.x; i < total; i += 256) {
    const int k = i / a.d, ch = i - k * a.d;
    const float2 f = part[(size_t)k * a.c + ch];
    q += (double)f.y + ((double)f.x - mean) * ((double)f.x - mean) * min(a.ppc, a.p - k * a.ppc);
  }
  const double var = block_sum(q, red) / m;
  if (threadIdx.x == 0) {
    a.mean[blockIdx.x] = (float)mean;
    a.rstd[blockIdx.x] = (float)(1.0 / sqrt(var + (double)a.eps));
  }
}

// ---- y = drop(act((x - mean) * rstd * gamma + beta)) ----
template <typename T, int V> __global__ __launch_bounds__(256) void norm_apply_kernel(const NormArgs a) {
  const NormTile t = NormTile::get<V>(a);
  if (!t.on) return;
  NormChan<V> ch;
  ch.load(a, t.img, t.c0, true);
#pragma unroll
  for (int e = 0; e < V; ++e) ch.rstd[e] *= ch.gamma[e];
  const uint64_t offset = a.drop.thresh ? drop_offset(a.drop) : 0;
  const T* x = (const T*)a.x + (size_t)t.img * a.p * a.xcs + t.c0;
  T* y = (T*)a.y + (size_t)t.img * a.p * a.ycs + t.c0;
  for (int p = t.p0 + t.row; p < t.p1; p += a.rows) {
    float v[V];
    load_v<T, V>(x + (size_t)p * a.xcs, v);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = (v[e] - ch.mean[e]) * ch.rstd[e] + ch.beta[e];
    act_apply<V>(v, a.act);
    if (a.drop.thresh) drop_apply<V>(v, ((uint64_t)t.img * a.p + p) * a.c + t.c0, a.drop, offset);
    store_v<T, V>(y + (size_t)p * a.ycs, v);
  }
}

// ---- backward, first half: (A, B) of every channel over a chunk ----
template <typename T, int V> __global__ __launch_bounds__(256) void norm_bwd_sums_kernel(const NormArgs a) {
  __shared__ float2 red[256 * V];
  const NormTile t = NormTile::get<V>(a);
  if (t.on) {
    NormChan<V> ch;
    ch.load(a, t.img, t.c0, true);
    const uint64_t offset = a.drop.thresh ? drop_offset(a.drop) : 0;
    float sa[V], sb[V];
#pragma unroll
    for (int e = 0; e < V; ++e) sa[e] = sb[e] = 0.f;
    const T* x = (const T*)a.x + (size_t)t.img * a.p * a.xcs + t.c0;
    const T* dy = (const T*)a.dy + (size_t)t.img * a.p * a.dycs + t.c0;
    for (int p = t.p0 + t.row; p < t.p1; p += a.rows) {
      float v[V], g[V];
      load_v<T, V>(x + (size_t)p * a.xcs, v);
      load_v<T, V>(dy + (size_t)p * a.dycs, g);
      if (a.drop.thresh) drop_apply<V>(g, ((uint64_t)t.img * a.p + p) * a.c + t.c0, a.drop, offset);
      norm_dz<V>(a, ch, v, g);
#pragma unroll
      for (int e = 0; e < V; ++e) { sa[e] += g[e]; sb[e] += g[e] * v[e]; }
    }
#pragma unroll
    for (int e = 0; e < V; ++e) red[threadIdx.x * V + e] = make_float2(sa[e], sb[e]);
  }
  __syncthreads();
  const int nch = min(a.cb * V, a.c - (int)blockIdx.y * a.cb * V);
  for (int k = threadIdx.x; k < nch; k += 256) {
    float2 s = make_float2(0.f, 0.f);
    for (int r = 0; r < a.rows; ++r) { const float2 f = red[r * a.cb * V + k]; s.x += f.x; s.y += f.y; }
    a.part[((size_t)t.img * a.chunks + t.chunk) * a.c + blockIdx.y * a.cb * V + k] = s;
  }
}

// ---- backward, join: one workgroup per (image, group): (A, B) of its channels over the chunks, then S1, S2 ----
__global__ __launch_bounds__(256) void norm_bwd_join_kernel(const NormArgs a) {
  __shared__ double2 sum[256];
  __shared__ double red[4];
  const int img = blockIdx.x / a.groups, g = blockIdx.x - img * a.groups;
  double s1 = 0.0, s2 = 0.0;
  for (int cb0 = 0; cb0 < a.d; cb0 += 256) {
    const int nd = min(256, a.d - cb0), lanes = 256 / nd, k0 = threadIdx.x / nd, ch = threadIdx.x - k0 * nd;
    double sa = 0.0, sb = 0.0;
    if (k0 < lanes)
      for (int k = k0; k < a.chunks; k += lanes) {
        const float2 f = a.part[((size_t)img * a.chunks + k) * a.c + (size_t)g * a.d + cb0 + ch];
        sa += f.x; sb += f.y;
      }
    __syncthreads();
    sum[threadIdx.x] = make_double2(sa, sb);
    __syncthreads();
    if ((int)threadIdx.x < nd) {
      sa = sb = 0.0;
      for (int k = 0; k < lanes; ++k) { sa += sum[k * nd + threadIdx.x].x; sb += sum[k * nd + threadIdx.x].y; }
      const int c = g * a.d + cb0 + threadIdx.x;
      a.ab[(size_t)img * a.c + c] = make_float2((float)sa, (float)sb);
      const double gm = a.gamma ? (double)a.gamma[c] : 1.0;
      s1 += gm * sa; s2 += gm * sb;
    }
  }
  const double m = (double)a.p * a.d;
  s1 = block_sum(s1, red); s2 = block_sum(s2, red);
  if (threadIdx.x == 0) a.s12[blockIdx.x] = make_float2((float)(s1 / m), (float)(s2 / m));
}

// ---- backward, second half: dx ----
template <typename T, int V> __global__ __launch_bounds__(256) void norm_bwd_apply_kernel(const NormArgs a) {
  const NormTile t = NormTile::get<V>(a);
  if (!t.on) return;
  NormChan<V> ch;
  ch.load(a, t.img, t.c0, true);
  float s1[V], s2[V];
#pragma unroll
  for (int e = 0; e < V; ++e) { const float2 s = a.s12[(size_t)t.img * a.groups + (t.c0 + e) / a.d]; s1[e] = s.x; s2[e] = s.y; }
  const uint64_t offset = a.drop.thresh ? drop_offset(a.drop) : 0;
  const T* x = (const T*)a.x + (size_t)t.img * a.p * a.xcs + t.c0;
  const T* dy = (const T*)a.dy + (size_t)t.img * a.p * a.dycs + t.c0;
  T* dx = (T*)a.y + (size_t)t.img * a.p * a.ycs + t.c0;
  for (int p = t.p0 + t.row; p < t.p1; p += a.rows) {
    float v[V], g[V];
    load_v<T, V>(x + (size_t)p * a.xcs, v);
    load_v<T, V>(dy + (size_t)p * a.dycs, g);
    if (a.drop.thresh) drop_apply<V>(g, ((uint64_t)t.img * a.p + p) * a.c + t.c0, a.drop, offset);
    norm_dz<V>(a, ch, v, g);
#pragma unroll
    for (int e = 0; e < V; ++e) g[e] = ch.rstd[e] * (g[e] * ch.gamma[e] - s1[e] - v[e] * s2[e]);
    store_v<T, V>(dx + (size_t)p * a.ycs, g);
  }
}

// ---- dropout: y = drop(x) [+ res]; a thread per generator block of eight elements ----
template <typename T, bool ALIGNED> __global__ __launch_bounds__(256) void dropout_kernel(const T* x, const T* res, T* y, size_t count, DropArgs d) {
  const size_t blocks = (count + 7) / 8, stride = (size_t)gridDim.x * 256;
  const uint64_t offset = d.thresh ? drop_offset(d) : 0;
  for (size_t b = (size_t)blockIdx.x * 256 + threadIdx.x; b < blocks; b += stride) {
    float v[8], r[8];
    if (ALIGNED && 8 * b + 8 <= count) {
      load_v<T, 8>(x + 8 * b, v);
      if (res) load_v<T, 8>(res + 8 * b, r);
      if (d.thresh) drop_apply<8>(v, 8 * b, d, offset);
      if (res)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += r[e];
      store_v<T, 8>(y + 8 * b, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 8 * b + e < count ? (float)x[8 * b + e] : 0.f;
      if (d.thresh) drop_apply<8>(v, 8 * b, d, offset);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (8 * b + e < count) y[8 * b + e] = (T)(res ? v[e] + (float)res[8 * b + e] : v[e]);
    }
  }
}

}  // namespace fisr
